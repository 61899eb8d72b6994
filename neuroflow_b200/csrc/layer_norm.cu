// layer_norm.cu -- layer norm over the last dimension of (rows, d), forward (into the
// input's type, or straight into FP8 groups of 128) and backward.
//
//   mu = sum x / d,  v = sum (x - mu)^2 / d,  r = 1 / sqrt(v + eps),  xh = (x - mu) r
//   y  = gamma xh + beta
//   a  = gamma dy,  dx = r (a - mean(a) - xh mean(a xh))
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// All statistics and sums are fp32; the variance is the mean of the centred squares (a
// second sweep), not E[x^2] - mu^2, which cancels when |mu| is large against the spread.
// Outputs are rounded once.
#include "block_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"

namespace nfx {
namespace {

constexpr int kAnyThreads = 256;

// Sum of v over the block, the same value in every thread.  `red` holds one float per warp.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();  // the previous sum has been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
    return t;
}

// Any width, alignment and stride: one block per row, the row read three times (from L2
// after the first).
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) norm_any_kernel(NormArgs a) {
    __shared__ float red[kAnyThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float fd = static_cast<float>(a.d);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        float s = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) s += to_f32(x[i]);
        const float mu = __fdiv_rn(block_sum(s, red), fd);
        s = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float c = to_f32(x[i]) - mu;
            s = fmaf(c, c, s);
        }
        const float rs = __frsqrt_rn(__fdiv_rn(block_sum(s, red), fd) + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mu;
            if (a.rstd) a.rstd[r] = rs;
        }
        auto out = [&](int i) {
            const float xh = (to_f32(x[i]) - mu) * rs;
            const float g = a.gamma ? load_any(a.gamma, a.ptype, i) : 1.0f;
            return fmaf(xh, g, a.beta ? load_any(a.beta, a.ptype, i) : 0.0f);
        };
        if (a.y) {
            T* y = static_cast<T*>(a.y) + r * a.ldy;
            for (int i = threadIdx.x; i < a.d; i += kAnyThreads) y[i] = from_f32<T>(out(i));
        } else {
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

// Any width: a block takes every gridDim.x-th row and adds its rows' parameter gradients,
// in their order, to its own two rows of partial sums (each column always by one thread).
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) norm_grad_any_kernel(NormGradArgs a) {
    __shared__ float red[kAnyThreads / 32];
    const float fd = static_cast<float>(a.d);
    float* pg = a.part + static_cast<int64_t>(blockIdx.x) * a.d;
    float* pb = a.part + (static_cast<int64_t>(a.parts) + blockIdx.x) * a.d;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
        const float mu = a.mean[r], rs = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float xh = (to_f32(x[i]) - mu) * rs, g = to_f32(dy[i]);
            const float ga = a.gamma ? g * load_any(a.gamma, a.ptype, i) : g;
            s1 += ga;
            s2 = fmaf(ga, xh, s2);
            if (a.part) {
                const bool first = r == blockIdx.x;
                pg[i] = fmaf(g, xh, first ? 0.0f : pg[i]);
                pb[i] = g + (first ? 0.0f : pb[i]);
            }
        }
        s1 = __fdiv_rn(block_sum(s1, red), fd);
        s2 = __fdiv_rn(block_sum(s2, red), fd);
        for (int i = threadIdx.x; i < a.d; i += kAnyThreads) {
            const float xh = (to_f32(x[i]) - mu) * rs, g = to_f32(dy[i]);
            const float ga = a.gamma ? g * load_any(a.gamma, a.ptype, i) : g;
            dx[i] = from_f32<T>(rs * (ga - s1 - xh * s2));
        }
    }
}

// 32 columns per block, 8 threads per column over the partial sums, joined in a fixed order.
__global__ void __launch_bounds__(256) column_reduce_kernel(const float* __restrict__ part, int parts,
                                                            int64_t n, void* out, int otype) {
    __shared__ float red[8][33];
    const int c = threadIdx.x & 31, t = threadIdx.x >> 5;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + c;
    float s = 0.0f;
    if (i < n)
        for (int p = t; p < parts; p += 8) s += part[p * n + i];
    red[t][c] = s;
    __syncthreads();
    if (t == 0 && i < n) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += red[k][c];
        store_any(out, otype, i, s);
    }
}

template <typename T>
cudaError_t norm_t(const NormArgs& a, cudaStream_t s) {
    const int64_t cap = 8ll * device_sm_count();
    norm_any_kernel<T><<<static_cast<int>(a.rows < cap ? a.rows : cap), kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t norm_grad_t(const NormGradArgs& a, cudaStream_t s) {
    if (a.rows > 0) norm_grad_any_kernel<T><<<a.parts, kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t layer_norm_launch(const NormArgs& a, int xtype, cudaStream_t s) {
    if (xtype == kF32) return norm_t<float>(a, s);
    if (xtype == kBF16) return norm_t<__nv_bfloat16>(a, s);
    return norm_t<__half>(a, s);
}

int layer_norm_parts(int64_t rows, int64_t) {
    const int64_t cap = 2ll * device_sm_count();
    return static_cast<int>(rows < cap ? rows : cap);
}

cudaError_t column_reduce_launch(const float* part, int parts, int64_t n, void* out, int otype,
                                 cudaStream_t s) {
    column_reduce_kernel<<<static_cast<unsigned>((n + 31) / 32), 256, 0, s>>>(part, parts, n, out, otype);
    return cudaGetLastError();
}

cudaError_t layer_norm_backward_launch(const NormGradArgs& a, int xtype, cudaStream_t s) {
    cudaError_t e = xtype == kF32    ? norm_grad_t<float>(a, s)
                    : xtype == kBF16 ? norm_grad_t<__nv_bfloat16>(a, s)
                                     : norm_grad_t<__half>(a, s);
    if (e == cudaSuccess && a.dgamma) e = column_reduce_launch(a.part, a.parts, a.d, a.dgamma, a.ptype, s);
    if (e == cudaSuccess && a.dbeta)
        e = column_reduce_launch(a.part + static_cast<int64_t>(a.parts) * a.d, a.parts, a.d, a.dbeta, a.ptype, s);
    return e;
}

}  // namespace nfx
