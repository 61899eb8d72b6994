// gemm_dense.cu -- product of two 16-bit matrices with bias, activation and residual in its epilogue, and the
// activation's gradient.
//
//   Z = A B^T + bias,  C = act(Z) + R;   dz = dy act'(z),  dbias = sum over rows of dz
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "dense_ops.h"
#include "nfx_internal.h"
#include "numerics.cuh"
#include "sm100.cuh"

namespace nfx {
namespace {

// GELU's tanh form is z s(2u), s the logistic function, u = sqrt(2 / pi) (z + 0.044715 z^3).  -2u, in units
// of log 2; where it is above kFar the value and the slope are under 2^-90 and are taken as zero.
constexpr float kFar = 100.0f;
__device__ __forceinline__ float gelu_exponent(float z) { return -2.302208198f * fmaf(z, (0.044715f * z) * z, z); }
__device__ __forceinline__ float act_of(float z, int act) {
    if (act == 1) {
        const float t = gelu_exponent(z), e = exp2f(fminf(t, kFar));
        return (t > kFar ? -0.0f : z) * __fdividef(1.0f, 1.0f + e);
    }
    return act == 2 ? relu_ref(z) : z;
}

constexpr int kT = 64, kTK = 16;

template <typename T>
__global__ void __launch_bounds__(256) gemm_simple_kernel(GemmDenseArgs p) {
    __shared__ float sa[kTK][kT + 1], sb[kTK][kT + 1];
    const T* A = static_cast<const T*>(p.A);
    const T* B = static_cast<const T*>(p.B);
    const int m0 = blockIdx.x * kT, n0 = blockIdx.y * kT, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    // pieces of 512 terms: one chain of roundings over a long K drifts
    float acc[4][4] = {}, total[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += kTK) {
        for (int e = threadIdx.x; e < kT * kTK; e += 256) {
            const int ra = p.a_t ? e % kT : e / kTK, ka = p.a_t ? e / kT : e % kTK;
            const int rb = p.b_t ? e % kT : e / kTK, kb = p.b_t ? e / kT : e % kTK;
            const int64_t ma = m0 + ra, nb = n0 + rb;
            sa[ka][ra] = ma < p.M && k0 + ka < p.K ? to_f32(A[p.a_t ? (k0 + ka) * p.lda + ma : ma * p.lda + k0 + ka]) : 0.0f;
            sb[kb][rb] = nb < p.N && k0 + kb < p.K ? to_f32(B[p.b_t ? (k0 + kb) * p.ldb + nb : nb * p.ldb + k0 + kb]) : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < kTK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
        if ((k0 + kTK) % 512 == 0 || k0 + kTK >= p.K)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) total[i][j] += acc[i][j], acc[i][j] = 0.0f;
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m >= p.M || n >= p.N) continue;
            float z = total[i][j];
            if (p.bias) z += load_any(p.bias, p.btype, n);
            if (p.Z) store_any(p.Z, p.ctype, m * p.ldz + n, z);
            z = act_of(z, p.act);
            if (p.res) z += load_any(p.res, p.ctype, m * p.ldres + n);
            store_any(p.C, p.ctype, m * p.ldc + n, z);
        }
}

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

int64_t gemm_dense_workspace(const void*, int64_t, int, const void*, int64_t, int, int64_t, int64_t, int64_t) { return 0; }

cudaError_t gemm_dense_launch(const GemmDenseArgs& p, cudaStream_t s) {
    const dim3 grid((p.M + kT - 1) / kT, (p.N + kT - 1) / kT);
    if (p.abtype == kBF16) gemm_simple_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else gemm_simple_kernel<__half><<<grid, 256, 0, s>>>(p);
    return cudaGetLastError();
}

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
