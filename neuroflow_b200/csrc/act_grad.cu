// act_grad.cu -- the activation's gradient and the bias gradient.
//
//   dz = dy act'(z),  dbias = sum over rows of dz (in fp32, before dz is rounded)
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ops.h"
#include "nfx_internal.h"

namespace nfx {
namespace {

// GELU's tanh form is z s(2u), s the logistic function, u = sqrt(2 / pi) (z + 0.044715 z^3).  -2u, in units
// of log 2; where it is above kFar the value and the slope are under 2^-90 and are taken as zero.
constexpr float kFar = 100.0f;
__device__ __forceinline__ float gelu_exponent(float z) { return -2.302208198f * fmaf(z, (0.044715f * z) * z, z); }

// The slope of the activation.  GELU's is s + z s (1 - s) (2u)', with 1 - s as e s, e = e^(-2u) (the
// difference would lose the digits that z (2u)' multiplies); beyond |z| = 30 it is 0 or 1.
__device__ __forceinline__ float slope_of(float z, int act) {
    if (act == 2) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if (act != 1) return 1.0f;
    const float c = fminf(fmaxf(z, -30.0f), 30.0f), t = gelu_exponent(c), e = exp2f(fminf(t, kFar)), s = __fdividef(1.0f, 1.0f + e);
    const float v = fmaf(c * s * (e * s), 1.5957691216057308f * fmaf(0.134145f * c, c, 1.0f), s);
    return z != z ? z : (t > kFar ? 0.0f : v);
}

// A block takes 256 columns of a share of the rows, one column a thread: the column's sum stays in a register.
template <typename T>
__global__ void __launch_bounds__(256) act_grad_kernel(ActGradArgs a) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t r0 = a.rows * blockIdx.y / gridDim.y, r1 = a.rows * (blockIdx.y + 1) / gridDim.y;
    if (c >= a.cols) return;
    float s = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        float v = to_f32(static_cast<const T*>(a.dy)[r * a.lddy + c]);
        if (a.act) v *= slope_of(to_f32(static_cast<const T*>(a.z)[r * a.ldz + c]), a.act);
        s += v;
        if (a.dz) static_cast<T*>(a.dz)[r * a.lddz + c] = from_f32<T>(v);
    }
    if (a.part) a.part[blockIdx.y * a.cols + c] = s;
}

}  // namespace

int act_grad_parts(int64_t rows, int64_t cols) {
    const int64_t want = (rows + 31) / 32;
    return static_cast<int>(want < 256 ? want : 256);
}

cudaError_t act_grad_launch(const ActGradArgs& a, int type, cudaStream_t s) {
    const dim3 grid(static_cast<unsigned>((a.cols + 255) / 256), a.parts);
    if (type == kF32) act_grad_kernel<float><<<grid, 256, 0, s>>>(a);
    else if (type == kBF16) act_grad_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
    else act_grad_kernel<__half><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace nfx
