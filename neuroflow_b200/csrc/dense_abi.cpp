// dense_abi.cpp -- extern "C" entry points of the RMS norm with residual, the 16-bit matrix product, the
// activation's gradient and gradient clipping (include/nfx.h): argument checks, then the launchers.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/nfx.h"
#include "dense_ops.h"
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
bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(n) == 0; }
bool el(const void* p, int type) { return aligned(p, nfx::type_bytes(type)); }

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

constexpr const char* kTypes = "a type must be NFX_F32, NFX_BF16 or NFX_F16";
constexpr const char* kUnaligned = "a pointer is not aligned to its element";
constexpr const char* kStride = "a row stride is smaller than its row";

// What the forms of the RMS norm share; nullptr when it is in order.
const char* rms_check(int64_t rows, int64_t d, int x_type, int h_type, int param_type, bool with_h) {
    if (!type_ok(x_type) || !type_ok(param_type) || (with_h && !type_ok(h_type))) return kTypes;
    if (rows < 0 || d < 1) return "rows must be >= 0 and d >= 1";
    // columns are 32-bit numbers, also when rounded up to a whole FP8 group; loops that step by more count without a sign
    if (d > kIntMax - 256) return "d must be below 2^31 - 256";
    if (with_h && h_type != x_type && h_type != NFX_F32) return "the residual must have x's type or be NFX_F32";
    return nullptr;
}

int rms_call(const char* fn, nfx::RmsArgs& a, const void* x, int x_type, int64_t ldx, const void* residual, int sum_type,
             int64_t ld_res, const void* gamma, int param_type, int64_t rows, int64_t d, float eps, void* sum, int64_t ld_sum,
             float* rstd, cudaStream_t s) {
    if (const char* w = rms_check(rows, d, x_type, sum_type, param_type, residual != nullptr)) return bad(fn, w);
    if (!(eps >= 0.0f)) return bad(fn, "eps must be >= 0");
    if (sum && !residual) return bad(fn, "a sum is written with a residual only");
    if (rows > 1 && (ldx < d || (residual && ld_res < d) || (sum && ld_sum < d))) return bad(fn, kStride);
    if (rows == 0) return NFX_OK;
    if (!x) return bad(fn, "null pointer");
    const int h_type = residual ? sum_type : x_type;
    if (!el(x, x_type) || !el(residual, h_type) || !el(sum, h_type) || !el(gamma, param_type) || !aligned(rstd, 4))
        return bad(fn, kUnaligned);
    a.x = x, a.ldx = ldx, a.res = residual, a.ldres = ld_res, a.gamma = gamma, a.ptype = param_type, a.rows = rows;
    a.d = static_cast<int>(d), a.eps = eps, a.sum = sum, a.ldsum = ld_sum, a.rstd = rstd;
    return launched(fn, nfx::rms_norm_launch(a, x_type, h_type, s));
}

int grad_list(const char* fn, std::vector<nfx::GradTensor>& list, const void* const* grads, const int64_t* counts, const int* types,
              void* const* out, const int* out_types, bool write, int64_t tensors) {
    if (tensors < 0 || tensors > kIntMax) return bad(fn, "tensors must be >= 0 and below 2^31");
    if (tensors > 0 && (!grads || !counts || !types || (out && !out_types))) return bad(fn, "null pointer");
    list.resize(static_cast<size_t>(tensors));
    for (int64_t i = 0; i < tensors; ++i) {
        nfx::GradTensor& t = list[static_cast<size_t>(i)];
        t.n = counts[i], t.src = grads[i], t.src_type = types[i];
        t.dst = !write ? nullptr : (out ? out[i] : const_cast<void*>(grads[i]));
        t.dst_type = out ? out_types[i] : types[i];
        if (t.n < 0) return bad(fn, "a count is negative");
        if (!type_ok(t.src_type) || (write && !type_ok(t.dst_type))) return bad(fn, kTypes);
        if (t.n > 0 && (!t.src || (write && !t.dst))) return bad(fn, "null pointer");
        if (!el(t.src, t.src_type) || (write && !el(t.dst, t.dst_type))) return bad(fn, kUnaligned);
    }
    return NFX_OK;
}

int workspace_check(const char* fn, const void* ws, int64_t have, int64_t need) {
    if (need > 0 && (!ws || have < need)) return bad(fn, "the workspace is smaller than the entry's _workspace says");
    if (need > 0 && !aligned(ws, 16)) return bad(fn, "the workspace must be 16-byte aligned");
    return NFX_OK;
}

}  // namespace

extern "C" {

int nfx_rms_norm(const void* x, int x_type, int64_t ldx, const void* residual, int sum_type, int64_t ld_residual, const void* gamma,
                 int param_type, int64_t rows, int64_t d, float eps, void* y, int64_t ldy, void* sum, int64_t ld_sum, float* rstd,
                 void* stream) {
    const char* fn = "nfx_rms_norm";
    return guarded(fn, [&]() -> int {
        if (rows > 1 && ldy < d) return bad(fn, kStride);
        if (rows > 0 && !y) return bad(fn, "null pointer");
        if (type_ok(x_type) && !el(y, x_type)) return bad(fn, kUnaligned);
        nfx::RmsArgs a{};
        a.y = y, a.ldy = ldy;
        return rms_call(fn, a, x, x_type, ldx, residual, sum_type, ld_residual, gamma, param_type, rows, d, eps, sum, ld_sum, rstd,
                        static_cast<cudaStream_t>(stream));
    });
}

int nfx_rms_norm_fp8(const void* x, int x_type, int64_t ldx, const void* residual, int sum_type, int64_t ld_residual,
                     const void* gamma, int param_type, int64_t rows, int64_t d, float eps, uint8_t* codes, int64_t ld_codes,
                     float* scales, int64_t scale_row_stride, int64_t scale_block_stride, void* sum, int64_t ld_sum, float* rstd,
                     void* stream) {
    const char* fn = "nfx_rms_norm_fp8";
    return guarded(fn, [&]() -> int {
        if (rows > 1 && ld_codes < d) return bad(fn, kStride);
        if (rows > 0 && (!codes || !scales)) return bad(fn, "null pointer");
        if (!aligned(scales, 4)) return bad(fn, kUnaligned);
        nfx::RmsArgs a{};
        a.q = {codes, ld_codes, scales, scale_row_stride, scale_block_stride};
        return rms_call(fn, a, x, x_type, ldx, residual, sum_type, ld_residual, gamma, param_type, rows, d, eps, sum, ld_sum, rstd,
                        static_cast<cudaStream_t>(stream));
    });
}

int64_t nfx_rms_norm_backward_workspace(int64_t rows, int64_t d) {
    if (rows <= 0 || d <= 0) return 0;
    return static_cast<int64_t>(nfx::rms_norm_parts(rows, d)) * d * 4;
}

int nfx_rms_norm_backward(const void* dy, int dy_type, int64_t lddy, const void* h, int h_type, int64_t ldh, const float* rstd,
                          const void* gamma, int param_type, const void* dsum, int64_t ld_dsum, int64_t rows, int64_t d, void* dx,
                          int64_t lddx, void* dres, int64_t ld_dres, void* dgamma, void* workspace, int64_t workspace_bytes,
                          void* stream) {
    const char* fn = "nfx_rms_norm_backward";
    return guarded(fn, [&]() -> int {
        if (const char* w = rms_check(rows, d, dy_type, h_type, param_type, true)) return bad(fn, w);
        if (rows > 1 && (lddy < d || ldh < d || (dsum && ld_dsum < d) || (dx && lddx < d) || (dres && ld_dres < d)))
            return bad(fn, kStride);
        if (rows > 0 && (!dy || !h || !rstd)) return bad(fn, "null pointer");
        if (!el(dy, dy_type) || !el(h, h_type) || !el(dsum, h_type) || !el(dx, dy_type) || !el(dres, h_type) ||
            !el(gamma, param_type) || !el(dgamma, param_type) || !aligned(rstd, 4))
            return bad(fn, kUnaligned);
        if (dgamma)
            if (const int rc = workspace_check(fn, workspace, workspace_bytes, nfx_rms_norm_backward_workspace(rows, d))) return rc;
        nfx::RmsGradArgs a{};
        a.dy = dy, a.lddy = lddy, a.h = h, a.ldh = ldh, a.rstd = rstd, a.gamma = gamma, a.ptype = param_type;
        a.dsum = dsum, a.lddsum = ld_dsum, a.rows = rows, a.d = static_cast<int>(d);
        a.dx = dx, a.lddx = lddx, a.dres = dres, a.lddres = ld_dres, a.dgamma = dgamma;
        a.parts = rows > 0 ? nfx::rms_norm_parts(rows, d) : 0;
        a.part = dgamma && rows > 0 ? static_cast<float*>(workspace) : nullptr;
        return launched(fn, nfx::rms_norm_backward_launch(a, dy_type, h_type, static_cast<cudaStream_t>(stream)));
    });
}

int64_t nfx_gemm_workspace(const void* A, int64_t lda, int a_trans, const void* B, int64_t ldb, int b_trans, int64_t M, int64_t N,
                           int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > kIntMax - 256 || N > kIntMax - 256 || K > kIntMax - 256) return 0;
    return nfx::gemm_dense_workspace(A, lda, a_trans, B, ldb, b_trans, M, N, K);
}

int nfx_gemm(const void* A, int64_t lda, int a_trans, const void* B, int64_t ldb, int b_trans, int ab_type, int64_t M, int64_t N,
             int64_t K, const void* bias, int bias_type, int act, const void* residual, int64_t ld_residual, void* C, int c_type,
             int64_t ldc, void* Z, int64_t ldz, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "nfx_gemm";
    return guarded(fn, [&]() -> int {
        if (M < 0 || N < 0 || K < 0) return bad(fn, "M, N and K must be >= 0");
        if (M > kIntMax - 256 || N > kIntMax - 256 || K > kIntMax - 256) return bad(fn, "M, N and K must be below 2^31 - 256");
        if (ab_type != NFX_BF16 && ab_type != NFX_F16) return bad(fn, "ab_type must be NFX_BF16 or NFX_F16");
        if (!type_ok(c_type) || !type_ok(bias_type)) return bad(fn, kTypes);
        if (c_type != ab_type && c_type != NFX_F32) return bad(fn, "c_type must be ab_type or NFX_F32");
        if (act < 0 || act > 2) return bad(fn, "act must be 0, 1 or 2");
        if ((a_trans != 0 && a_trans != 1) || (b_trans != 0 && b_trans != 1)) return bad(fn, "a_trans and b_trans must be 0 or 1");
        if (M == 0 || N == 0) return NFX_OK;
        if (!C || (K > 0 && (!A || !B))) return bad(fn, "null pointer");
        // a matrix of one row has no row stride to speak of
        const int64_t ra = a_trans ? K : M, ca = a_trans ? M : K, rb = b_trans ? K : N, cb = b_trans ? N : K;
        if ((ra > 1 && lda < ca) || (rb > 1 && ldb < cb) || (M > 1 && (ldc < N || (residual && ld_residual < N) || (Z && ldz < N))))
            return bad(fn, kStride);
        if (!el(A, ab_type) || !el(B, ab_type) || !el(bias, bias_type) || !el(residual, c_type) || !el(C, c_type) || !el(Z, c_type))
            return bad(fn, kUnaligned);
        if (((M + 127) / 128) * ((N + 15) / 16) > kIntMax / 16) return bad(fn, "too many tiles");
        nfx::GemmDenseArgs p{};
        p.A = A, p.lda = ra > 1 ? lda : ca, p.a_t = a_trans, p.B = B, p.ldb = rb > 1 ? ldb : cb, p.b_t = b_trans, p.abtype = ab_type;
        p.M = static_cast<int>(M), p.N = static_cast<int>(N), p.K = static_cast<int>(K);
        p.bias = bias, p.btype = bias_type, p.act = act, p.res = residual, p.ldres = M > 1 ? ld_residual : N;
        p.C = C, p.ctype = c_type, p.ldc = M > 1 ? ldc : N, p.Z = Z, p.ldz = M > 1 ? ldz : N;
        if (const int rc = workspace_check(fn, workspace, workspace_bytes, nfx_gemm_workspace(A, lda, a_trans, B, ldb, b_trans, M, N, K)))
            return rc;
        p.ws = workspace;
        p.err = nfx::device_error_word();
        if (!p.err) return nfx::set_thread_error(NFX_INTERNAL, "nfx_gemm: cannot allocate the device error word");
        return launched(fn, nfx::gemm_dense_launch(p, static_cast<cudaStream_t>(stream)));
    });
}

void nfx_debug_gemm_plan(int64_t M, int64_t N, int64_t K, int a_trans, int b_trans, int aligned, int sms, int* columns, int* split,
                         int* deep, int* runs) {
    const void* at = reinterpret_cast<const void*>(static_cast<uintptr_t>(aligned ? 16 : 2));
    const int64_t n = sms < 1 ? 1 : sms;
    if (nfx::few_rows(at, 8, a_trans, at, 8, b_trans, M, N, K)) {
        *columns = -1, *split = nfx::gemm_few_split(M, N, K, b_trans, n), *deep = 0, *runs = 1;
        return;
    }
    const nfx::DensePlan c = nfx::gemm_dense_plan(M, N, K, a_trans, n);
    *columns = c.columns, *split = c.split, *deep = c.deep, *runs = c.runs;
}

int64_t nfx_act_backward_workspace(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return static_cast<int64_t>(nfx::act_grad_parts(rows, cols)) * cols * 4;
}

int nfx_act_backward(const void* dy, int64_t lddy, const void* z, int64_t ldz, int type, int act, int64_t rows, int64_t cols, void* dz,
                     int64_t lddz, void* dbias, int bias_type, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "nfx_act_backward";
    return guarded(fn, [&]() -> int {
        if (!type_ok(type) || !type_ok(bias_type)) return bad(fn, kTypes);
        if (act < 0 || act > 2) return bad(fn, "act must be 0, 1 or 2");
        if (rows < 0 || cols < 0) return bad(fn, "rows and cols must be >= 0");
        if (rows > kIntMax || cols > kIntMax) return bad(fn, "rows and cols must be below 2^31");
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        nfx::ActGradArgs a{};
        if (rows > 0 && cols > 0) {
            if (!dy || (act && !z)) return bad(fn, "null pointer");
            if (rows > 1 && (lddy < cols || (act && ldz < cols) || (dz && lddz < cols))) return bad(fn, kStride);
            if (!el(dy, type) || !el(z, type) || !el(dz, type) || !el(dbias, bias_type)) return bad(fn, kUnaligned);
            if (dbias)
                if (const int rc = workspace_check(fn, workspace, workspace_bytes, nfx_act_backward_workspace(rows, cols))) return rc;
            a.dy = dy, a.lddy = lddy, a.z = z, a.ldz = ldz, a.act = act, a.rows = rows, a.cols = cols, a.dz = dz, a.lddz = lddz;
            a.parts = nfx::act_grad_parts(rows, cols);
            a.part = dbias ? static_cast<float*>(workspace) : nullptr;
            if (dz || dbias)
                if (const int rc = launched(fn, nfx::act_grad_launch(a, type, st))) return rc;
        }
        if (dbias && cols > 0) return launched(fn, nfx::column_reduce_launch(a.part, a.parts, cols, dbias, nullptr, bias_type, st));
        return NFX_OK;
    });
}

int64_t nfx_grad_norm_workspace(int64_t tensors) { return tensors < 0 ? 0 : 8 * nfx::grad_norm_partials(tensors); }

int nfx_grad_norm(const void* const* grads, const int64_t* counts, const int* types, int64_t tensors, float* norm, void* workspace,
                  int64_t workspace_bytes, void* stream) {
    const char* fn = "nfx_grad_norm";
    return guarded(fn, [&]() -> int {
        std::vector<nfx::GradTensor> list;
        if (const int rc = grad_list(fn, list, grads, counts, types, nullptr, nullptr, false, tensors)) return rc;
        if (!norm) return bad(fn, "null pointer");
        if (!aligned(norm, 4)) return bad(fn, kUnaligned);
        if (const int rc = workspace_check(fn, workspace, workspace_bytes, nfx_grad_norm_workspace(tensors))) return rc;
        return launched(fn, nfx::grad_norm_launch(list.data(), tensors, static_cast<double*>(workspace), norm,
                                                  static_cast<cudaStream_t>(stream)));
    });
}

int nfx_clip_grad_norm(const void* const* grads, const int64_t* counts, const int* types, void* const* out, const int* out_types,
                       int64_t tensors, double max_norm, double eps, float* norm, void* workspace, int64_t workspace_bytes,
                       void* stream) {
    const char* fn = "nfx_clip_grad_norm";
    return guarded(fn, [&]() -> int {
        if (!(max_norm >= 0.0)) return bad(fn, "max_norm must be >= 0");
        if (!(eps >= 0.0) || std::isinf(eps)) return bad(fn, "eps must be >= 0 and finite");
        std::vector<nfx::GradTensor> list;
        if (const int rc = grad_list(fn, list, grads, counts, types, out, out_types, true, tensors)) return rc;
        if (!norm) return bad(fn, "null pointer");
        if (!aligned(norm, 4)) return bad(fn, kUnaligned);
        if (const int rc = workspace_check(fn, workspace, workspace_bytes, nfx_grad_norm_workspace(tensors))) return rc;
        return launched(fn, nfx::grad_clip_launch(list.data(), tensors, static_cast<double*>(workspace), max_norm, eps, norm,
                                                  static_cast<cudaStream_t>(stream)));
    });
}

}  // extern "C"
