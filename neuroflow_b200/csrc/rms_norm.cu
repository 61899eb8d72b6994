// rms_norm.cu -- root-mean-square norm over the last dimension of (rows, d) with the residual's addition,
// forward (into the input's type, or straight into FP8 groups of 128) and backward.
//
//   h = x + res, rounded to the residual's type;  r = 1 / sqrt(sum h^2 / d + eps)
//   y = h r gamma
//   a = gamma dy,  xh = h r,  dh = r (a - xh mean(a xh)) + dsum
//   dgamma = sum over rows of dy xh
//
// The norm is that of the sum as it is stored, so the backward pass, which reads the stored sum, is the
// gradient of exactly what was computed.  All sums are fp32.
#include "dense_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "row_pack.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

constexpr int kAnyThreads = 256;

// The sum of `a` over the block, the same bits in every thread.  `red` holds one number per warp.
__device__ __forceinline__ float block_sum(float a, float* red) {
    a = warp_sum(a);
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    float t = 0.0f;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
    return t;
}

// Any width: one block per row, the row read twice (from L2 the second time).
template <typename T, typename H>
__global__ void __launch_bounds__(kAnyThreads) rms_any_kernel(RmsArgs a) {
    __shared__ float red[kAnyThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const H* res = a.res ? static_cast<const H*>(a.res) + r * a.ldres : nullptr;
        H* sum = a.sum ? static_cast<H*>(a.sum) + r * a.ldsum : nullptr;
        // (the sum may be written over x or the residual: the second sweep reads it, by the same threads)
        float s = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            float h = to_f32(x[i]);
            if (res) {
                const H hr = from_f32<H>(h + to_f32(res[i]));
                h = to_f32(hr);
                if (sum) sum[i] = hr;
            }
            s = fmaf(h, h, s);
        }
        const float rs = __frsqrt_rn(__fdiv_rn(block_sum(s, red), static_cast<float>(a.d)) + a.eps);
        if (threadIdx.x == 0 && a.rstd) a.rstd[r] = rs;
        auto out = [&](int i) {
            float h;
            if (sum) h = to_f32(sum[i]);
            else if (res) h = to_f32(from_f32<H>(to_f32(x[i]) + to_f32(res[i])));
            else h = to_f32(x[i]);
            return (h * rs) * (a.gamma ? load_any(a.gamma, a.ptype, i) : 1.0f);
        };
        if (a.y) {
            T* y = static_cast<T*>(a.y) + r * a.ldy;
            for (int i = threadIdx.x; i < a.d; i += kAnyThreads) y[i] = from_f32<T>(out(i));
        } else {
            if (sum) __syncthreads();  // the groups below are read by other threads than wrote the sum
            const int blocks = (a.d + kGroup - 1) / kGroup;
            for (int b = warp; b < blocks; b += kAnyThreads / 32) {
                float v[kGroup / 32], am = 0.0f;
#pragma unroll
                for (int j = 0; j < kGroup / 32; ++j) {
                    const int i = b * kGroup + j * 32 + lane;
                    v[j] = i < a.d ? out(i) : 0.0f;
                    am = fmaxf(am, finite_abs(v[j]));
                }
                const float sc = group_scale(warp_max(am)), inv = __frcp_rn(sc);
#pragma unroll
                for (int j = 0; j < kGroup / 32; ++j) {
                    const int i = b * kGroup + j * 32 + lane;
                    if (i < a.d) a.q.codes[r * a.q.ld + i] = static_cast<uint8_t>(e4m3_code(v[j], inv));
                }
                if (lane == 0) a.q.scales[r * a.q.srs + b * a.q.sbs] = sc;
            }
        }
    }
}

// Any width: a block takes every gridDim.x-th row and adds its rows' parameter gradients, in their order,
// to its own row of partial sums (each column always by one thread).
template <typename T, typename H>
__global__ void __launch_bounds__(kAnyThreads) rms_grad_any_kernel(RmsGradArgs a) {
    __shared__ float red[kAnyThreads / 32];
    float* pg = a.part + static_cast<int64_t>(blockIdx.x) * a.d;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        const H* h = static_cast<const H*>(a.h) + r * a.ldh;
        const H* ds = a.dsum ? static_cast<const H*>(a.dsum) + r * a.lddsum : nullptr;
        const float rs = a.rstd[r];
        float s = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float xh = to_f32(h[i]) * rs, g = to_f32(dy[i]);
            s = fmaf(a.gamma ? g * load_any(a.gamma, a.ptype, i) : g, xh, s);
            if (a.part) pg[i] = fmaf(g, xh, r == blockIdx.x ? 0.0f : pg[i]);
        }
        s = __fdiv_rn(block_sum(s, red), static_cast<float>(a.d));
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float xh = to_f32(h[i]) * rs, g = to_f32(dy[i]);
            float o = rs * fmaf(-xh, s, a.gamma ? g * load_any(a.gamma, a.ptype, i) : g);
            if (ds) o += to_f32(ds[i]);
            if (a.dx) static_cast<T*>(a.dx)[r * a.lddx + i] = from_f32<T>(o);
            if (a.dres) static_cast<H*>(a.dres)[r * a.lddres + i] = from_f32<H>(o);
        }
    }
}

template <typename T, typename H>
cudaError_t rms_t(const RmsArgs& a, cudaStream_t s) {
    const int64_t cap = 8ll * device_sm_count();
    rms_any_kernel<T, H><<<static_cast<int>(a.rows < cap ? a.rows : cap), kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, typename H>
cudaError_t rms_grad_t(RmsGradArgs& a, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    rms_grad_any_kernel<T, H><<<a.parts, kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t rms_norm_launch(const RmsArgs& a, int xtype, int htype, cudaStream_t s) {
    if (xtype == kF32) return rms_t<float, float>(a, s);
    if (xtype == kBF16) return htype == kF32 ? rms_t<__nv_bfloat16, float>(a, s) : rms_t<__nv_bfloat16, __nv_bfloat16>(a, s);
    return htype == kF32 ? rms_t<__half, float>(a, s) : rms_t<__half, __half>(a, s);
}

int rms_norm_parts(int64_t rows, int64_t d) {
    const int64_t cap = 4ll * device_sm_count();
    return static_cast<int>(rows < cap ? rows : cap);
}

cudaError_t rms_norm_backward_launch(const RmsGradArgs& args, int dytype, int htype, cudaStream_t s) {
    RmsGradArgs a = args;
    cudaError_t e;
    if (dytype == kF32) e = rms_grad_t<float, float>(a, s);
    else if (dytype == kBF16) e = htype == kF32 ? rms_grad_t<__nv_bfloat16, float>(a, s) : rms_grad_t<__nv_bfloat16, __nv_bfloat16>(a, s);
    else e = htype == kF32 ? rms_grad_t<__half, float>(a, s) : rms_grad_t<__half, __half>(a, s);
    if (e == cudaSuccess && a.dgamma) e = column_reduce_launch(a.part, a.parts, a.d, a.dgamma, nullptr, a.ptype, s);
    return e;
}

}  // namespace nfx
