// act_grad.cu -- the activation's gradient and the bias gradient.
//
//   dz = dy act'(z),  dbias = sum over rows of dz (in fp32, before dz is rounded)
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ops.h"
#include "nfx_internal.h"
#include "rms_parts.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

// GELU's tanh form is z s(2u), s the logistic function, u = sqrt(2 / pi) (z + 0.044715 z^3).  -2u, in units
// of log 2; where it is above kFar the value and the slope are under 2^-90 and are taken as zero.
constexpr float kFar = 100.0f;
__device__ __forceinline__ float gelu_exponent(float z) { return -2.302208198f * fmaf(z, (0.044715f * z) * z, z); }

// The slope of the activation.  GELU's is s + z s (1 - s) (2u)', with 1 - s as e s, e = e^(-2u) (the
// difference would lose the digits that z (2u)' multiplies); beyond |z| = 30 it is 0 or 1.  The hardware's
// exponential and reciprocal are a few 2^-22 off.
__device__ __forceinline__ float slope_of(float z, int act) {
    if (act == 2) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if (act != 1) return 1.0f;
    const float c = fminf(fmaxf(z, -30.0f), 30.0f), t = gelu_exponent(c);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(t, kFar)));
    const float s = __fdividef(1.0f, 1.0f + e);
    const float v = fmaf(c * s * (e * s), fmaf(1.5957691216057308f * 0.134145f * c, c, 1.5957691216057308f), s);
    return z != z ? z : (t > kFar ? 0.0f : v);
}

// A warp takes 32 VE columns (by 16-byte words; single ones, four a lane, where rows are not aligned to them) of every
// eighth row of the block's share, two rows at a time; the columns' sums stay in registers and are joined over the
// block's warps at the end.  4095x2048 bf16 with GELU and the bias gradient: see gemm_dense.cu's training step.
constexpr int kWarps = 8;

template <typename T, int VE, int VPT>
__global__ void __launch_bounds__(32 * kWarps, 4) act_grad_kernel(ActGradArgs a) {
    constexpr int E = VE * VPT, kU = 2;
    __shared__ float joined[kWarps][32 * E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32 * E + lane * VE;
    const int64_t r0 = a.rows * blockIdx.y / gridDim.y, r1 = a.rows * (blockIdx.y + 1) / gridDim.y;
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
    for (int64_t r = r0 + warp; r < r1; r += kWarps * kU) {
        Elems<T, VE> y[kU][VPT], z[kU][VPT];
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int64_t c = c0 + j * 32 * VE, row = r + u * kWarps;
                if (row < r1 && c < a.cols) {
                    y[u][j].load(static_cast<const T*>(a.dy) + row * a.lddy + c);
                    if (a.act) z[u][j].load(static_cast<const T*>(a.z) + row * a.ldz + c);
                } else {
                    y[u][j].zero(), z[u][j].zero();
                }
            }
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int64_t c = c0 + j * 32 * VE, row = r + u * kWarps;
                if (row >= r1 || c >= a.cols) continue;
                float v[VE];
                y[u][j].get(v);
                if (a.act) {
#pragma unroll
                    for (int i = 0; i < VE; ++i) v[i] *= slope_of(z[u][j].at(i), a.act);
                }
#pragma unroll
                for (int i = 0; i < VE; ++i) s[j * VE + i] += v[i];
                if (a.dz) {
                    Elems<T, VE> o;
                    o.set(v);
                    o.store(static_cast<T*>(a.dz) + row * a.lddz + c);
                }
            }
    }
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < E; ++e) joined[warp][e * 32 + lane] = s[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * E; i += 32 * kWarps) {
        float t = joined[0][i];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) t += joined[w][i];
        const int e = i / 32, l = i % 32;
        const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 * E + (e / VE * 32 + l) * VE + e % VE;
        if (c < a.cols) a.part[blockIdx.y * a.cols + c] = t;
    }
}

template <typename T, int VE, int VPT>
cudaError_t act_grad_go(const ActGradArgs& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.cols + 32 * VE * VPT - 1) / (32 * VE * VPT)), static_cast<unsigned>(a.parts));
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, act_grad_kernel<T, VE, VPT>, a);
}

template <typename T>
cudaError_t act_grad_t(const ActGradArgs& a, cudaStream_t s) {
    constexpr int VE = 16 / sizeof(T);
    const auto on16 = [&](const void* p, int64_t ld) { return !p || aligned_rows(p, a.rows, ld, sizeof(T), 16); };
    if (a.cols % VE == 0 && on16(a.dy, a.lddy) && (!a.act || on16(a.z, a.ldz)) && on16(a.dz, a.lddz)) return act_grad_go<T, VE, 1>(a, s);
    return act_grad_go<T, 1, 4>(a, s);
}

}  // namespace

// Shares of the rows: enough to fill the SMs, each of 32 rows at least.
int act_grad_parts(int64_t rows, int64_t cols) {
    const int64_t across = (cols + 255) / 256, all = (4ll * device_sm_count() + across - 1) / across, want = (rows + 31) / 32;
    const int64_t n = want < all ? want : all;
    return static_cast<int>(n < 1 ? 1 : n);
}

cudaError_t act_grad_launch(const ActGradArgs& a, int type, cudaStream_t s) {
    if (type == kF32) return act_grad_t<float>(a, s);
    return type == kBF16 ? act_grad_t<__nv_bfloat16>(a, s) : act_grad_t<__half>(a, s);
}

}  // namespace nfx
