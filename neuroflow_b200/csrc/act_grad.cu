// act_grad.cu -- the activation's gradient and the bias gradient.
//
//   dz = dy act'(z),  dbias = sum over rows of dz (in fp32, before dz is rounded)
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "rms_parts.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

// The activation's slope at two numbers.  GELU's tanh form is z s(2u), s the logistic function, u = sqrt(2 / pi) (z +
// 0.044715 z^3), and its slope s + z s (1 - s) (2u)', with 1 - s as e s, e = e^(-2u) (the difference would lose the
// digits that z (2u)' multiplies).  Beyond |z| = 30, and where e is over 2^60, it is 0 or 1 to 2^-50.  Two numbers
// share a reciprocal and the packed products; the hardware's exponential and reciprocal are a few 2^-22 off.
constexpr float kFar = 60.0f;
__device__ __forceinline__ float2 slope2(float2 z, int act) {
    if (act == 2) return make_float2(z.x > 0.0f ? 1.0f : (z.x != z.x ? z.x : 0.0f), z.y > 0.0f ? 1.0f : (z.y != z.y ? z.y : 0.0f));
    const auto both = [](float v) { return make_float2(v, v); };
    const float2 c = make_float2(fminf(fmaxf(z.x, -30.0f), 30.0f), fminf(fmaxf(z.y, -30.0f), 30.0f)), c2 = mul2_rn(c, c);
    // -2u in units of log 2, and (2u)'
    const float2 t = mul2_rn(c, fma2_rn(c2, both(-2.302208198f * 0.044715f), both(-2.302208198f)));
    const float2 d = fma2_rn(c2, both(1.5957691216057308f * 0.134145f), both(1.5957691216057308f));
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(fminf(t.x, kFar)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(fminf(t.y, kFar)));
    const float a = 1.0f + e.x, b = 1.0f + e.y, r = __fdividef(1.0f, a * b);
    const float2 s = mul2_rn(both(r), make_float2(b, a));
    const float2 v = fma2_rn(mul2_rn(mul2_rn(c, s), mul2_rn(e, s)), d, s);
    return make_float2(z.x != z.x ? z.x : (t.x > kFar ? 0.0f : v.x), z.y != z.y ? z.y : (t.y > kFar ? 0.0f : v.y));
}

// A warp takes 32 VE columns (by 16-byte words; single ones, four a lane, where rows are not aligned to them) of every
// eighth row of the block's share, the next row on its way while one is worked on; the columns' sums stay in
// registers and are joined over the block's warps at the end.  16384x4096 bf16 with GELU and the bias gradient:
// 70 us, 5.8 TB/s (two rows at a time without a next one 88 us, with one, which spills, 104); 16384x4095, by single
// elements, 103 us; 4095x2048: 12.8 us, of which joining the shares takes 2.6.
constexpr int kWarps = 8;

template <typename T, int VE, int VPT>
__global__ void __launch_bounds__(32 * kWarps, 4) act_grad_kernel(ActGradArgs a) {
    constexpr int E = VE * VPT;
    __shared__ float joined[kWarps][32 * E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32 * E + lane * VE;
    const int64_t r0 = a.rows * blockIdx.y / gridDim.y, r1 = a.rows * (blockIdx.y + 1) / gridDim.y;
    grid_dep_launch();
    grid_dep_wait();  // what the kernel before this one wrote may be read from here on
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
    Elems<T, VE> ny[VPT], nz[VPT];
    const auto fetch = [&](int64_t r) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int64_t c = c0 + j * 32 * VE;
            if (r < r1 && c < a.cols) {
                ny[j].load(static_cast<const T*>(a.dy) + r * a.lddy + c);
                if (a.act) nz[j].load(static_cast<const T*>(a.z) + r * a.ldz + c);
            } else {
                ny[j].zero(), nz[j].zero();
            }
        }
    };
    fetch(r0 + warp);
    for (int64_t r = r0 + warp; r < r1; r += kWarps) {
        Elems<T, VE> y[VPT], z[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) y[j] = ny[j], z[j] = nz[j];
        fetch(r + kWarps);
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = y[e / VE].at(e % VE);
        if (a.act) {
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 w = slope2(make_float2(z[e / VE].at(e % VE), z[(e + 1) / VE].at((e + 1) % VE)), a.act);
                v[e] *= w.x, v[e + 1] *= w.y;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += v[e];
        if (!a.dz) continue;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int64_t c = c0 + j * 32 * VE;
            if (c >= a.cols) continue;
            float o[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) o[i] = v[j * VE + i];
            Elems<T, VE> w;
            w.set(o);
            w.store(static_cast<T*>(a.dz) + r * a.lddz + c);
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
