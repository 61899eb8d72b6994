// dense_ops.h -- the operators of a pre-norm block in 16 bits (RMS norm with the residual's addition, the
// matrix product with bias, activation and residual, the activation's gradient, gradient clipping):
// arguments and launchers shared by the kernels and the C-ABI layer (dense_abi.cpp).  Sizes are checked by
// the C-ABI layer.
#pragma once

#include "block_ops.h"

namespace nfx {

struct RmsArgs {
    const void* x;
    int64_t ldx;
    const void* res;  // added to x, or nullptr
    int64_t ldres;
    const void* gamma;  // (d,) or nullptr (ones)
    int ptype;
    int64_t rows;
    int d;
    float eps;
    void* y;  // (rows, d) of x's type, or nullptr: the FP8 form
    int64_t ldy;
    Fp8Out q;
    void* sum;  // x + res in res's type, or nullptr
    int64_t ldsum;
    float* rstd;  // (rows,) or nullptr
};
// htype: the type of res and sum (x's own where there is none)
cudaError_t rms_norm_launch(const RmsArgs& a, int xtype, int htype, cudaStream_t s);

struct RmsGradArgs {
    const void* dy;
    int64_t lddy;
    const void* h;
    int64_t ldh;
    const float* rstd;
    const void* gamma;  // (d,) or nullptr (ones)
    int ptype;
    const void* dsum;  // gradient that reaches h otherwise, of h's type, or nullptr
    int64_t lddsum;
    int64_t rows;
    int d;
    void* dx;  // of dy's type, or nullptr
    int64_t lddx;
    void* dres;  // of h's type, or nullptr
    int64_t lddres;
    void* dgamma;  // (d,) of ptype, or nullptr
    float* part;   // parts x d partial sums, or nullptr
    int parts;
};
int rms_norm_parts(int64_t rows, int64_t d);
cudaError_t rms_norm_backward_launch(const RmsGradArgs& a, int dytype, int htype, cudaStream_t s);

struct GemmDenseArgs {
    const void* A;  // (M, K): element (m, k) at m lda + k, or at k lda + m with a_t
    int64_t lda;
    int a_t;
    const void* B;  // (N, K), the same
    int64_t ldb;
    int b_t;
    int abtype;  // kBF16 or kF16
    int M, N, K;
    const void* bias;  // (N,) or nullptr
    int btype;
    int act;  // 0 none, 1 GELU (tanh form), 2 ReLU
    const void* res;  // (M, N) of C's type, or nullptr
    int64_t ldres;
    void* C;
    int ctype;
    int64_t ldc;
    void* Z;  // what the activation is taken of, of C's type, or nullptr
    int64_t ldz;
    void* ws;  // room for operands that TMA cannot read and for sums of runs of K, gemm_dense_workspace bytes
    int runs;  // set by the launcher
    unsigned* err;
    unsigned long long wait_ns;
};
// whether TMA reads a matrix of 16-bit elements: `rows` contiguous runs, `ld` from one to the next
inline bool tma_operand(const void* p, int64_t ld, int64_t rows) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || ld % 8 == 0);
}
// Whether a product is the kernel's for few rows (gemm_few.cu): up to 16 of them (16x4096x4096: 10.0 us, 10.6 with the
// narrow kernel; 32x4096x4096: 13.7, 10.8), and up to 32 with rows of B that TMA cannot read, which would be copied
// first (32x1023x1023: 6.9, 7.3).
inline bool few_rows(const void* A, int64_t lda, int a_t, const void* B, int64_t ldb, int b_t, int64_t M, int64_t N, int64_t K) {
    if (a_t || M > 32) return false;
    return M <= 16 || (!b_t && !(tma_operand(A, lda, M) && tma_operand(B, ldb, N)));
}
int gemm_few_split(int64_t M, int64_t N, int64_t K, int b_t, int64_t sms);
cudaError_t gemm_few_launch(const GemmDenseArgs& a, int split, cudaStream_t s);
// how a product is cut on `sms` SMs: rows of A to a tile of the narrow kernel (0: the kernel of CTA pairs),
// CTAs that share K, whether the narrow kernel takes an SM's memory for one CTA's ring, and runs of K that are joined
// by a second kernel
struct DensePlan {
    int columns, split;
    bool deep;
    int runs;
};
DensePlan gemm_dense_plan(int64_t M, int64_t N, int64_t K, int a_t, int64_t sms);
int64_t gemm_dense_workspace(const void* A, int64_t lda, int a_t, const void* B, int64_t ldb, int b_t, int64_t M, int64_t N, int64_t K);
cudaError_t gemm_dense_launch(const GemmDenseArgs& a, cudaStream_t s);

struct ActGradArgs {
    const void* dy;
    int64_t lddy;
    const void* z;  // nullptr without an activation
    int64_t ldz;
    int act;
    int64_t rows, cols;
    void* dz;  // or nullptr
    int64_t lddz;
    float* part;  // parts x cols partial sums, or nullptr
    int parts;
};
int act_grad_parts(int64_t rows, int64_t cols);
cudaError_t act_grad_launch(const ActGradArgs& a, int type, cudaStream_t s);

struct GradTensor {
    const void* src;
    void* dst;  // nullptr: the norm only
    int64_t n;
    int src_type, dst_type;
};
int64_t grad_norm_partials(int64_t tensors);
cudaError_t grad_norm_launch(const GradTensor* t, int64_t tensors, double* part, float* norm, cudaStream_t s);
cudaError_t grad_clip_launch(const GradTensor* t, int64_t tensors, double* part, double max_norm, double eps, float* norm,
                             cudaStream_t s);

}  // namespace nfx
