// rms_norm_grad.cu -- gradient of the RMS norm, joined with the one that reaches its input from elsewhere.
//
//   a = gamma dy,  xh = h r,  dh = r (a - xh mean(a xh)) + dsum
//   dgamma = sum over rows of dy xh
//
// All sums are fp32.
#include <atomic>

#include "dense_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "rms_parts.cuh"
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
cudaError_t rms_grad_t(RmsGradArgs& a, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    rms_grad_any_kernel<T, H><<<a.parts, kAnyThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

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
