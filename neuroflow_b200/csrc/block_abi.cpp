// block_abi.cpp -- extern "C" entry points of the layer norm, the FP8 block quantiser and the
// FP8 block-scaled product (include/nfx.h): argument checks, then the launchers.
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/nfx.h"
#include "block_ops.h"
#include "nfx_internal.h"

namespace nfx {
int set_thread_error(int code, const std::string& msg);
}

namespace {

constexpr int64_t kIntMax = 0x7FFFFFFF;

int bad(const char* fn, const char* what) {
    return nfx::set_thread_error(NFX_INVALID_ARG, std::string(fn) + ": " + what);
}
int launched(const char* fn, cudaError_t e) {
    if (e == cudaSuccess) return NFX_OK;
    return nfx::set_thread_error(NFX_INTERNAL, std::string(fn) + ": launch failed: " + cudaGetErrorString(e));
}
bool type_ok(int t) { return t == NFX_F32 || t == NFX_BF16 || t == NFX_F16; }
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(n) == 0; }

// The checks that layer norm's forms share; nullptr when they pass.
const char* norm_check(int x_type, int param_type, int64_t rows, int64_t d, int64_t ldx, const void* x) {
    if (!type_ok(x_type)) return "x_type must be NFX_F32, NFX_BF16 or NFX_F16";
    if (!type_ok(param_type)) return "param_type must be NFX_F32, NFX_BF16 or NFX_F16";
    if (rows < 0 || d < 1) return "rows must be >= 0 and d >= 1";
    // the kernels for any width add 256 to a 32-bit column index before they compare it with d
    if (d > kIntMax - 256) return "d must be below 2^31 - 256";
    if (rows > 1 && ldx < d) return "a row stride is smaller than d";
    if (rows > 0 && !x) return "null pointer";
    return nullptr;
}
bool elements_aligned(const void* p, int type) { return aligned(p, nfx::type_bytes(type)); }

int norm_call(const char* fn, const nfx::NormArgs& a, int x_type, cudaStream_t s) {
    if (a.rows == 0) return NFX_OK;
    if (!elements_aligned(a.x, x_type) || !elements_aligned(a.gamma, a.ptype) || !elements_aligned(a.beta, a.ptype) ||
        !aligned(a.mean, 4) || !aligned(a.rstd, 4))
        return bad(fn, "a pointer is not aligned to its element");
    return launched(fn, nfx::layer_norm_launch(a, x_type, s));
}

// C entries answer with a status; nothing is thrown through them.
template <typename F>
int guarded(const char* fn, F f) {
    try {
        return f();
    } catch (...) {
        try {
            return nfx::set_thread_error(NFX_INTERNAL, std::string(fn) + ": out of host memory");
        } catch (...) {
            return NFX_INTERNAL;
        }
    }
}

}  // namespace

extern "C" {

int nfx_layer_norm(const void* x, int x_type, int64_t ldx, const void* gamma, const void* beta, int param_type,
                   int64_t rows, int64_t d, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                   void* stream) {
    const char* fn = "nfx_layer_norm";
    return guarded(fn, [&]() -> int {
        if (const char* w = norm_check(x_type, param_type, rows, d, ldx, x)) return bad(fn, w);
        if (!(eps >= 0.0f)) return bad(fn, "eps must be >= 0");
        if (rows > 1 && ldy < d) return bad(fn, "a row stride is smaller than d");
        if (rows > 0 && !y) return bad(fn, "null pointer");
        if (!elements_aligned(y, x_type)) return bad(fn, "a pointer is not aligned to its element");
        nfx::NormArgs a{};
        a.x = x, a.ldx = ldx, a.gamma = gamma, a.beta = beta, a.ptype = param_type, a.rows = rows;
        a.d = static_cast<int>(d), a.eps = eps, a.y = y, a.ldy = ldy, a.mean = mean, a.rstd = rstd;
        return norm_call(fn, a, x_type, static_cast<cudaStream_t>(stream));
    });
}

int nfx_layer_norm_fp8(const void* x, int x_type, int64_t ldx, const void* gamma, const void* beta,
                       int param_type, int64_t rows, int64_t d, float eps, uint8_t* codes, int64_t ld_codes,
                       float* scales, int64_t scale_row_stride, int64_t scale_block_stride, float* mean,
                       float* rstd, void* stream) {
    const char* fn = "nfx_layer_norm_fp8";
    return guarded(fn, [&]() -> int {
        if (const char* w = norm_check(x_type, param_type, rows, d, ldx, x)) return bad(fn, w);
        if (!(eps >= 0.0f)) return bad(fn, "eps must be >= 0");
        if (rows > 1 && ld_codes < d) return bad(fn, "a row stride is smaller than d");
        if (rows > 0 && (!codes || !scales)) return bad(fn, "null pointer");
        if (!aligned(scales, 4)) return bad(fn, "a pointer is not aligned to its element");
        nfx::NormArgs a{};
        a.x = x, a.ldx = ldx, a.gamma = gamma, a.beta = beta, a.ptype = param_type, a.rows = rows;
        a.d = static_cast<int>(d), a.eps = eps, a.mean = mean, a.rstd = rstd;
        a.q = {codes, ld_codes, scales, scale_row_stride, scale_block_stride};
        return norm_call(fn, a, x_type, static_cast<cudaStream_t>(stream));
    });
}

int64_t nfx_layer_norm_backward_workspace(int64_t rows, int64_t d) {
    if (rows <= 0 || d <= 0) return 0;
    return 2 * static_cast<int64_t>(nfx::layer_norm_parts(rows, d)) * d * 4;
}

int nfx_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, int x_type,
                            const float* mean, const float* rstd, const void* gamma, int param_type,
                            int64_t rows, int64_t d, void* dx, int64_t lddx, void* dgamma, void* dbeta,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "nfx_layer_norm_backward";
    return guarded(fn, [&]() -> int {
        if (const char* w = norm_check(x_type, param_type, rows, d, ldx, x)) return bad(fn, w);
        if (rows > 1 && (lddy < d || lddx < d)) return bad(fn, "a row stride is smaller than d");
        if (rows > 0 && (!dy || !mean || !rstd || !dx)) return bad(fn, "null pointer");
        if (!elements_aligned(x, x_type) || !elements_aligned(dy, x_type) || !elements_aligned(dx, x_type) ||
            !elements_aligned(gamma, param_type) || !elements_aligned(dgamma, param_type) ||
            !elements_aligned(dbeta, param_type) || !aligned(mean, 4) || !aligned(rstd, 4))
            return bad(fn, "a pointer is not aligned to its element");
        const bool params = dgamma || dbeta;
        if (params && rows > 0) {
            if (!workspace || workspace_bytes < nfx_layer_norm_backward_workspace(rows, d))
                return bad(fn, "the workspace is smaller than nfx_layer_norm_backward_workspace says");
            if (!aligned(workspace, 16)) return bad(fn, "the workspace must be 16-byte aligned");
        }
        nfx::NormGradArgs a{};
        a.dy = dy, a.lddy = lddy, a.x = x, a.ldx = ldx, a.mean = mean, a.rstd = rstd, a.gamma = gamma;
        a.ptype = param_type, a.rows = rows, a.d = static_cast<int>(d), a.dx = dx, a.lddx = lddx;
        a.dgamma = dgamma, a.dbeta = dbeta;
        a.parts = rows > 0 ? nfx::layer_norm_parts(rows, d) : 0;
        a.part = params && rows > 0 ? static_cast<float*>(workspace) : nullptr;
        return launched(fn, nfx::layer_norm_backward_launch(a, x_type, static_cast<cudaStream_t>(stream)));
    });
}

int64_t nfx_fp8_quantise_workspace(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return up(rows, nfx::kGroup) * cols * 4;
}

int nfx_fp8_quantise(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t cols, int tile,
                     uint8_t* codes, int64_t ld_codes, float* scales, int64_t scale_row_stride,
                     int64_t scale_block_stride, uint8_t* codes_t, int64_t ld_codes_t, float* scales_t,
                     int64_t scale_t_row_stride, int64_t scale_t_block_stride, void* col_sums, int sums_type,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "nfx_fp8_quantise";
    return guarded(fn, [&]() -> int {
        if (!type_ok(x_type)) return bad(fn, "x_type must be NFX_F32, NFX_BF16 or NFX_F16");
        if (!type_ok(sums_type)) return bad(fn, "sums_type must be NFX_F32, NFX_BF16 or NFX_F16");
        if (rows < 0 || cols < 0) return bad(fn, "rows and cols must be >= 0");
        if (rows > kIntMax || cols > kIntMax) return bad(fn, "rows and cols must be below 2^31");
        if (tile != 0 && tile != 1) return bad(fn, "tile must be 0 or 1");
        if (tile && col_sums) return bad(fn, "column sums are made with groups of 1 x 128 only");
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (rows > 0 && cols > 0) {
            if (!x || !codes || !scales || (codes_t && !scales_t)) return bad(fn, "null pointer");
            if ((rows > 1 && (ldx < cols || ld_codes < cols)) || (codes_t && cols > 1 && ld_codes_t < rows))
                return bad(fn, "a row stride is smaller than its row");
            if (!elements_aligned(x, x_type) || !aligned(scales, 4) || !aligned(scales_t, 4) ||
                !elements_aligned(col_sums, sums_type))
                return bad(fn, "a pointer is not aligned to its element");
            if (up(rows, nfx::kGroup) * up(cols, nfx::kGroup) > kIntMax) return bad(fn, "too many blocks");
            if (col_sums) {
                if (!workspace || workspace_bytes < nfx_fp8_quantise_workspace(rows, cols))
                    return bad(fn, "the workspace is smaller than nfx_fp8_quantise_workspace says");
                if (!aligned(workspace, 16)) return bad(fn, "the workspace must be 16-byte aligned");
            }
            nfx::QuantArgs a{};
            a.x = x, a.ldx = ldx, a.rows = rows, a.cols = cols, a.tile = tile;
            a.q = {codes, ld_codes, scales, scale_row_stride, scale_block_stride};
            a.qt = {codes_t, ld_codes_t, scales_t, scale_t_row_stride, scale_t_block_stride};
            a.part = col_sums ? static_cast<float*>(workspace) : nullptr;
            if (const int rc = launched(fn, nfx::fp8_quantise_launch(a, x_type, st))) return rc;
        }
        if (col_sums && cols > 0)
            return launched(fn, nfx::column_reduce_launch(static_cast<float*>(workspace),
                                                          static_cast<int>(up(rows, nfx::kGroup)), cols, col_sums,
                                                          nullptr, sums_type, st));
        return NFX_OK;
    });
}

int nfx_fp8_gemm(const uint8_t* A, int64_t lda, const float* scale_a, int64_t scale_a_row_stride,
                 int64_t scale_a_block_stride, int a_tile, const uint8_t* B, int64_t ldb, const float* scale_b,
                 int64_t scale_b_row_stride, int64_t scale_b_block_stride, int b_tile, int64_t M, int64_t N,
                 int64_t K, const void* bias, int bias_type, int act, void* C, int c_type, int64_t ldc,
                 void* stream) {
    const char* fn = "nfx_fp8_gemm";
    return guarded(fn, [&]() -> int {
        if (M < 0 || N < 0 || K < 0) return bad(fn, "M, N and K must be >= 0");
        if (M > kIntMax - 256 || N > kIntMax - 256 || K > kIntMax - 256) return bad(fn, "M, N and K must be below 2^31 - 256");
        if (act < 0 || act > 2) return bad(fn, "act must be 0, 1 or 2");
        if (!type_ok(c_type) || !type_ok(bias_type)) return bad(fn, "a type must be NFX_F32, NFX_BF16 or NFX_F16");
        if ((a_tile != 0 && a_tile != 1) || (b_tile != 0 && b_tile != 1)) return bad(fn, "a_tile and b_tile must be 0 or 1");
        if (M == 0 || N == 0) return NFX_OK;
        if (!C || (K > 0 && (!A || !B || !scale_a || !scale_b))) return bad(fn, "null pointer");
        if (M > 1 && ldc < N) return bad(fn, "ldc is smaller than N");
        if (!elements_aligned(C, c_type) || !elements_aligned(bias, bias_type) || !aligned(scale_a, 4) || !aligned(scale_b, 4))
            return bad(fn, "a pointer is not aligned to its element");
        // a matrix of one row has no row stride to speak of
        const int64_t la = M > 1 ? lda : up(K, 16) * 16, lb = N > 1 ? ldb : up(K, 16) * 16;
        if (K > 0) {
            if (la < K || lb < K) return bad(fn, "a row stride is smaller than K");
            if (!aligned(A, 16) || !aligned(B, 16) || la % 16 || lb % 16)
                return bad(fn, "the rows of A and B must start on 16-byte boundaries");
        }
        if (up(M, 128) * up(N, 128) > kIntMax / 2) return bad(fn, "too many tiles");
        nfx::Fp8GemmArgs p{};
        p.A = A, p.lda = la, p.sa = scale_a, p.sars = scale_a_row_stride, p.sabs = scale_a_block_stride, p.a_tile = a_tile;
        p.B = B, p.ldb = lb, p.sb = scale_b, p.sbrs = scale_b_row_stride, p.sbbs = scale_b_block_stride, p.b_tile = b_tile;
        p.bias = bias, p.btype = bias_type, p.act = act, p.C = C, p.ctype = c_type, p.ldc = ldc;
        p.M = static_cast<int>(M), p.N = static_cast<int>(N), p.K = static_cast<int>(K);
        p.err = nfx::device_error_word();
        if (!p.err) return nfx::set_thread_error(NFX_INTERNAL, "nfx_fp8_gemm: cannot allocate the device error word");
        return launched(fn, nfx::fp8_gemm_launch(p, static_cast<cudaStream_t>(stream)));
    });
}

void nfx_debug_fp8_gemm_plan(int64_t M, int64_t N, int64_t K, int b_tile, int sms, int* columns, int* split, int* deep) {
    const nfx::Fp8Plan c = nfx::fp8_gemm_plan(M, N, K, b_tile, sms < 1 ? 1 : sms);
    *columns = c.columns, *split = c.split, *deep = c.deep;
}

}  // extern "C"
