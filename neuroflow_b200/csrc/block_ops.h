// block_ops.h -- the operators of one pre-norm FP8 linear layer (layer norm, the FP8
// block quantiser, the FP8 block-scaled product): arguments and launchers shared by the
// kernels and the C-ABI layer (block_abi.cpp).  Sizes are checked by the C-ABI layer.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace nfx {

// element types of the C-ABI (NFX_F32, NFX_BF16, NFX_F16)
enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline int64_t type_bytes(int t) { return t == kF32 ? 4 : 2; }

constexpr int kGroup = 128;         // elements that share one FP8 scale along K
constexpr float kE4m3Max = 448.0f;  // largest finite E4M3 value
constexpr float kMinScale = 0x1p-126f;

// FP8 codes with one scale per group: scale of (row r, block b) at r * row_stride + b * block_stride
struct Fp8Out {
    uint8_t* codes;
    int64_t ld;
    float* scales;
    int64_t srs, sbs;
};

struct NormArgs {
    const void* x;
    int64_t ldx;
    const void* gamma;  // (d,) or nullptr (ones)
    const void* beta;   // (d,) or nullptr (zeros)
    int ptype;          // type of gamma and beta
    int64_t rows;
    int d;
    float eps;
    void* y;  // (rows, d) of x's type, or nullptr: the FP8 form
    int64_t ldy;
    Fp8Out q;
    float* mean;  // (rows,) or nullptr
    float* rstd;
};
cudaError_t layer_norm_launch(const NormArgs& a, int xtype, cudaStream_t s);

struct NormGradArgs {
    const void* dy;
    int64_t lddy;
    const void* x;
    int64_t ldx;
    const float* mean;
    const float* rstd;
    const void* gamma;  // (d,) or nullptr (ones)
    int ptype;
    int64_t rows;
    int d;
    void* dx;
    int64_t lddx;
    void* dgamma;  // (d,) of ptype, or nullptr
    void* dbeta;
    float* part;  // 2 x parts x d partial sums
    int parts;
};
// how many partial sums of the parameter gradients a launch makes
int layer_norm_parts(int64_t rows, int64_t d);
cudaError_t layer_norm_backward_launch(const NormGradArgs& a, int xtype, cudaStream_t s);

// out0[i] = sum over p < parts of part[p * n + i], always in the same order (out of type otype); out1
// the same of the next parts * n numbers.  Either may be nullptr.
cudaError_t column_reduce_launch(const float* part, int parts, int64_t n, void* out0, void* out1, int otype,
                                 cudaStream_t s);

struct QuantArgs {
    const void* x;
    int64_t ldx;
    int64_t rows, cols;
    int tile;       // 0: groups of 1 x 128, 1: tiles of 128 x 128
    Fp8Out q;       // (rows, cols)
    Fp8Out qt;      // the transpose (cols, rows), or codes == nullptr
    float* part;    // (ceil(rows / 128), cols) column sums, or nullptr
};
cudaError_t fp8_quantise_launch(const QuantArgs& a, int xtype, cudaStream_t s);

struct Fp8GemmArgs {
    const uint8_t* A;  // (M, K)
    int64_t lda;
    const float* sa;
    int64_t sars, sabs;
    int a_tile;
    const uint8_t* B;  // (N, K)
    int64_t ldb;
    const float* sb;
    int64_t sbrs, sbbs;
    int b_tile;
    const void* bias;  // (N,) or nullptr
    int btype;
    int act;  // 0 none, 1 GELU (tanh form), 2 ReLU
    void* C;
    int ctype;
    int64_t ldc;
    int tma_c;  // set by the launcher: C's rows allow TMA stores
    int M, N, K;
    unsigned* err;
    unsigned long long wait_ns;
};
// how a product is cut on `sms` SMs: rows of A to a tile of the narrow kernel (0: the kernel of CTA pairs),
// CTAs that share K, and whether the narrow kernel takes an SM's memory for one CTA's ring
struct Fp8Plan {
    int columns, split;
    bool deep;
};
Fp8Plan fp8_gemm_plan(int64_t M, int64_t N, int64_t K, int b_tile, int64_t sms);
cudaError_t fp8_gemm_launch(const Fp8GemmArgs& a, cudaStream_t s);

#ifdef __CUDACC__
// ---- typed loads and stores -----------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// element i of an array whose type is known at run time
__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    if (type == kF32) return __ldg(static_cast<const float*>(p) + i);
    if (type == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, int64_t i, float v) {
    if (type == kF32) static_cast<float*>(p)[i] = v;
    else if (type == kBF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

// |v| for a group's maximum: infinities and NaN do not set a scale (they are encoded as
// +-448 and NaN), so one bad element leaves the rest of its group as it was.
__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;
}
// the scale of a group with maximum `amax`: amax / 448 rounded to fp32, at least 2^-126 so
// that its reciprocal is finite (a group of zeros has that scale)
__device__ __forceinline__ float group_scale(float amax) {
    return fmaxf(__fdiv_rn(amax, kE4m3Max), kMinScale);
}
#endif

}  // namespace nfx
