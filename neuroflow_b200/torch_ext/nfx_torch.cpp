// nfx_torch.cpp -- the torch front-end of the transformer-layer operators of libnfx.so (layer norm, FP8
// block quantiser, FP8 block-scaled product; in nfx_torch_dense.h those of a block in 16 bits): checks of the
// tensors, allocation of the outputs on the current stream, and the C-ABI call, in compiled code because a
// call on one token takes the GPU a few microseconds and the same steps in Python ten or more.
// neuroflow_b200/ops.py is the public face.
//
// Refused arguments raise neuroflow_b200._nfx.NfxError with status 1 (InvalidArg) before anything is
// launched; errors of the C-ABI raise it with theirs.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "nfx.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kGroup = 128;

[[noreturn]] void raise(int code, const std::string& msg) {
    py::gil_scoped_acquire gil;  // (a backward pass runs without it)
    py::object cls = py::module_::import("neuroflow_b200._nfx").attr("NfxError");
    py::object err = cls(code, msg);
    PyErr_SetObject(cls.ptr(), err.ptr());
    throw py::error_already_set();
}
[[noreturn]] void refuse(const char* fn, const std::string& what) { raise(NFX_INVALID_ARG, std::string(fn) + ": " + what); }
void check(int rc) {
    if (rc != NFX_OK) raise(rc, nfx_last_error());
}
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

int type_of(at::ScalarType t) {
    if (t == at::kFloat) return NFX_F32;
    if (t == at::kBFloat16) return NFX_BF16;
    return t == at::kHalf ? NFX_F16 : -1;
}
int type_of(const char* fn, const char* name, const Tensor& t) {
    if (!t.is_cuda()) refuse(fn, std::string(name) + " must be a CUDA tensor");
    const int k = type_of(t.scalar_type());
    if (k < 0) refuse(fn, std::string(name) + " must be float32, bfloat16 or float16, not " + c10::toString(t.scalar_type()));
    return k;
}
void same_device(const char* fn, const Tensor& x, const char* name, const Tensor& t) {
    if (t.device() != x.device()) refuse(fn, std::string(name) + " is on " + t.device().str() + ", not on " + x.device().str());
}

// A tensor as rows of its last dimension with one stride between them, without a copy.
struct Rows {
    int64_t rows, cols, ld;
};
Rows rows_of(const char* fn, const char* name, const Tensor& t) {
    const int64_t n = t.dim();
    if (n < 1) refuse(fn, std::string(name) + " needs at least one dimension");
    Rows r{1, t.size(n - 1), 0};
    int64_t expect = -1;  // the stride that the next outer dimension must have
    for (int64_t i = n - 2; i >= 0; --i) {
        const int64_t size = t.size(i);
        if (size != 1 && t.numel() > 0) {
            if (expect < 0) r.ld = t.stride(i);
            else if (t.stride(i) != expect)
                refuse(fn, "the rows of " + std::string(name) + " are not evenly strided: pass a contiguous tensor");
            expect = t.stride(i) * size;
        }
        r.rows *= size;
    }
    if (expect < 0) r.ld = r.cols;  // one row, or none
    if (t.numel() > 0) {
        if (r.cols > 1 && t.stride(n - 1) != 1) refuse(fn, "the last dimension of " + std::string(name) + " must be contiguous");
        if (r.rows > 1 && r.ld < r.cols) refuse(fn, "the rows of " + std::string(name) + " overlap");
    }
    return r;
}

const void* vector_of(const char* fn, const char* name, const OptTensor& t, int64_t n, const Tensor& x, int* type) {
    if (!t) return nullptr;
    *type = type_of(fn, name, *t);
    if (t->dim() != 1 || t->size(0) != n || (n > 1 && t->stride(0) != 1))
        refuse(fn, std::string(name) + " must be a contiguous vector of " + std::to_string(n));
    same_device(fn, x, name, *t);
    return t->const_data_ptr();
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) {
    return at::detail::empty_cuda(sizes, t, like.device(), std::nullopt);
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// `out` is written by the kernels, which autograd does not see.
void no_grad_out(const char* fn, const OptTensor& out) {
    if (out && out->requires_grad() && at::GradMode::is_enabled()) refuse(fn, "out must not be a tensor that requires grad");
}
// A call has written into its `out`: a backward pass that saved the buffer finds out by its version.
void written(const OptTensor& out) {
    if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

// Codes whose rows start on 16-byte boundaries, and scales with the block index outermost (the order in
// which the product reads them).
struct Fp8 {
    Tensor codes, scales;
    int64_t ld, srows;
    Fp8(int64_t rows, int64_t cols, int64_t scale_rows, const Tensor& like) : srows(scale_rows) {
        ld = up(cols > 0 ? cols : 1, 16) * 16;
        const int64_t stride[2] = {ld, 1}, sstride[2] = {1, scale_rows};
        codes = empty({rows, ld}, at::kFloat8_e4m3fn, like);
        if (ld != cols) codes = codes.as_strided({rows, cols}, stride);
        scales = at::detail::empty_strided_cuda({scale_rows, up(cols, kGroup)}, sstride, at::kFloat, like.device());
    }
    uint8_t* data() const { return static_cast<uint8_t*>(codes.data_ptr()); }
    float* scale() const { return static_cast<float*>(scales.data_ptr()); }
};

struct Norm {
    Rows x;
    int xt, pt = NFX_F32;
    const void *g, *b;
};
Norm norm_of(const char* fn, const Tensor& x, const OptTensor& gamma, const OptTensor& beta) {
    Norm n;
    n.xt = type_of(fn, "x", x);
    n.x = rows_of(fn, "x", x);
    if (n.x.cols < 1) refuse(fn, "the last dimension is empty");
    int gt = -1, bt = -1;
    n.g = vector_of(fn, "gamma", gamma, n.x.cols, x, &gt);
    n.b = vector_of(fn, "beta", beta, n.x.cols, x, &bt);
    if (gt >= 0 && bt >= 0 && gt != bt) refuse(fn, "beta must have gamma's type");
    n.pt = gt >= 0 ? gt : (bt >= 0 ? bt : static_cast<int>(NFX_F32));
    return n;
}
// mean and 1/std, one number for each row of x
std::pair<Tensor, Tensor> stats_of(const Tensor& x) {
    const auto sizes = x.sizes().slice(0, x.dim() - 1);
    return {empty(sizes, at::kFloat, x), empty(sizes, at::kFloat, x)};
}
float* ptr(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

struct NormOut {
    Tensor y, mean, rstd;
};
NormOut layer_norm(const Tensor& x, const OptTensor& gamma, const OptTensor& beta, double eps, const OptTensor& out, bool stats) {
    const char* fn = "layer_norm";
    const Norm n = norm_of(fn, x, gamma, beta);
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y;
    int64_t ldy = n.x.cols;
    if (out) {
        y = *out;
        if (y.sizes() != x.sizes() || y.scalar_type() != x.scalar_type() || y.device() != x.device())
            refuse(fn, "out must have x's shape, type and device");
        ldy = rows_of(fn, "out", y).ld;
        // (rows are read and written by different blocks; x itself is fine, its rows are read before they are written)
        if (at::get_overlap_status(x, y) == at::MemOverlapStatus::Partial) refuse(fn, "out shares a part of x's memory");
        no_grad_out(fn, out);
    } else {
        y = empty(x.sizes(), x.scalar_type(), x);
    }
    std::pair<Tensor, Tensor> st;
    if (stats) st = stats_of(x);
    check(nfx_layer_norm(x.const_data_ptr(), n.xt, n.x.ld, n.g, n.b, n.pt, n.x.rows, n.x.cols, static_cast<float>(eps),
                         y.data_ptr(), ldy, ptr(st.first), ptr(st.second), stream_of(x)));
    written(out);
    return {y, st.first, st.second};
}

py::object layer_norm_fp8(const Tensor& x, const OptTensor& gamma, const OptTensor& beta, double eps, bool stats) {
    const Norm n = norm_of("layer_norm_fp8", x, gamma, beta);
    c10::cuda::CUDAGuard guard(x.device());
    const Fp8 q(n.x.rows, n.x.cols, n.x.rows, x);
    std::pair<Tensor, Tensor> st;
    if (stats) st = stats_of(x);
    check(nfx_layer_norm_fp8(x.const_data_ptr(), n.xt, n.x.ld, n.g, n.b, n.pt, n.x.rows, n.x.cols, static_cast<float>(eps),
                             q.data(), q.ld, q.scale(), 1, q.srows, ptr(st.first), ptr(st.second), stream_of(x)));
    if (!stats) return py::make_tuple(q.codes, q.scales);
    return py::make_tuple(q.codes, q.scales, st.first, st.second);
}

struct NormGrad {
    Tensor dx, dgamma, dbeta;
};
NormGrad layer_norm_backward(const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd, const OptTensor& gamma,
                              bool param_grads) {
    const char* fn = "layer_norm_backward";
    const Norm n = norm_of(fn, x, gamma, std::nullopt);
    if (type_of(fn, "dy", dy) != n.xt || dy.sizes() != x.sizes()) refuse(fn, "dy must have x's shape and type");
    const Rows rdy = rows_of(fn, "dy", dy);
    same_device(fn, x, "dy", dy);
    for (const auto& p : {std::make_pair("mean", &mean), std::make_pair("rstd", &rstd)}) {
        if (type_of(fn, p.first, *p.second) != NFX_F32 || p.second->numel() != n.x.rows || !p.second->is_contiguous())
            refuse(fn, std::string(p.first) + " must be a contiguous float32 tensor of " + std::to_string(n.x.rows));
        same_device(fn, x, p.first, *p.second);
    }
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t d = n.x.cols;
    const Tensor dx = empty(x.sizes(), x.scalar_type(), x);
    Tensor dg, db, ws;
    int64_t bytes = 0;
    if (param_grads) {
        const at::ScalarType pt = gamma ? gamma->scalar_type() : at::kFloat;
        dg = empty({d}, pt, x);
        db = empty({d}, pt, x);
        bytes = nfx_layer_norm_backward_workspace(n.x.rows, d);
        ws = empty({bytes}, at::kByte, x);
    }
    check(nfx_layer_norm_backward(dy.const_data_ptr(), rdy.ld, x.const_data_ptr(), n.x.ld, n.xt,
                                  static_cast<const float*>(mean.const_data_ptr()), static_cast<const float*>(rstd.const_data_ptr()),
                                  n.g, n.pt, n.x.rows, d, dx.data_ptr(), d, param_grads ? dg.data_ptr() : nullptr,
                                  param_grads ? db.data_ptr() : nullptr, param_grads ? ws.data_ptr() : nullptr, bytes, stream_of(x)));
    return {dx, dg, db};
}

struct Quantised {
    Fp8 q;
    std::optional<Fp8> qt;
    Tensor sums;
};
Quantised fp8_quantise(const Tensor& x, bool tile, bool transposed, bool col_sums, at::ScalarType sums_type = at::kFloat) {
    const char* fn = "fp8_quantise";
    const int xt = type_of(fn, "x", x);
    const Rows r = rows_of(fn, "x", x);
    if (tile && col_sums) refuse(fn, "column sums are made with groups of 1 x 128 only");
    c10::cuda::CUDAGuard guard(x.device());
    const Fp8 q(r.rows, r.cols, tile ? up(r.rows, kGroup) : r.rows, x);
    std::optional<Fp8> qt;
    if (transposed) qt.emplace(r.cols, r.rows, tile ? up(r.cols, kGroup) : r.cols, x);
    Tensor sums, ws;
    int64_t bytes = 0;
    if (col_sums) {
        sums = empty({r.cols}, sums_type, x);
        bytes = nfx_fp8_quantise_workspace(r.rows, r.cols);
        ws = empty({bytes}, at::kByte, x);
    }
    check(nfx_fp8_quantise(x.const_data_ptr(), xt, r.ld, r.rows, r.cols, tile, q.data(), q.ld, q.scale(), 1, q.srows,
                           qt ? qt->data() : nullptr, qt ? qt->ld : 0, qt ? qt->scale() : nullptr, 1, qt ? qt->srows : 0,
                           col_sums ? sums.data_ptr() : nullptr, type_of(sums_type), col_sums ? ws.data_ptr() : nullptr, bytes,
                           stream_of(x)));
    return {q, qt, sums};
}

struct Operand {
    int64_t rows, k, ld, srs, sbs;
    const uint8_t* codes;
    const float* scales;
};
Operand operand_of(const char* fn, const char* name, const Tensor& c, const Tensor& s, bool tile) {
    if (!c.is_cuda() || c.dim() != 2 || (c.scalar_type() != at::kFloat8_e4m3fn && c.scalar_type() != at::kByte))
        refuse(fn, "the codes of " + std::string(name) + " must be a 2-D CUDA tensor of float8_e4m3fn (or its bytes)");
    const int64_t r = c.size(0), k = c.size(1);
    if (k > 1 && c.stride(1) != 1) refuse(fn, "the last dimension of " + std::string(name) + "'s codes must be contiguous");
    const int64_t sr = tile ? up(r, kGroup) : r, sk = up(k, kGroup);
    if (!s.is_cuda() || s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != sr || s.size(1) != sk || s.device() != c.device())
        refuse(fn, "the scales of " + std::string(name) + " must be float32 (" + std::to_string(sr) + ", " + std::to_string(sk) +
                       ") on " + c.device().str());
    return {r, k, c.stride(0), s.stride(0), s.stride(1), static_cast<const uint8_t*>(c.const_data_ptr()),
            static_cast<const float*>(s.const_data_ptr())};
}

Tensor fp8_gemm(const Tensor& ac, const Tensor& as, bool a_tile, const Tensor& bc, const Tensor& bs, bool b_tile,
                const OptTensor& bias, int64_t act, at::ScalarType out_dtype, const OptTensor& out) {
    const char* fn = "fp8_gemm";
    const Operand a = operand_of(fn, "a", ac, as, a_tile), b = operand_of(fn, "b", bc, bs, b_tile);
    if (a.k != b.k) refuse(fn, "a has " + std::to_string(a.k) + " columns and b " + std::to_string(b.k));
    same_device(fn, ac, "b", bc);
    if (act < 0 || act > 2) refuse(fn, "act must be 0, 1 or 2");
    int bt = NFX_F32;
    const void* bp = vector_of(fn, "bias", bias, b.rows, ac, &bt);
    Tensor c;
    int64_t ldc = b.rows;
    if (out) {
        c = *out;
        type_of(fn, "out", c);
        same_device(fn, ac, "out", c);
        if (c.dim() != 2 || c.size(0) != a.rows || c.size(1) != b.rows)
            refuse(fn, "out must be (" + std::to_string(a.rows) + ", " + std::to_string(b.rows) + ")");
        ldc = rows_of(fn, "out", c).ld;
        no_grad_out(fn, out);
    } else if (type_of(out_dtype) < 0) {
        refuse(fn, std::string("out_dtype must be float32, bfloat16 or float16, not ") + c10::toString(out_dtype));
    }
    c10::cuda::CUDAGuard guard(ac.device());
    if (!out) c = empty({a.rows, b.rows}, out_dtype, ac);
    check(nfx_fp8_gemm(a.codes, a.ld, a.scales, a.srs, a.sbs, a_tile, b.codes, b.ld, b.scales, b.srs, b.sbs, b_tile, a.rows, b.rows,
                       a.k, bp, bt, static_cast<int>(act), c.data_ptr(), type_of(c.scalar_type()), ldc, stream_of(ac)));
    written(out);
    return c;
}

// ---- autograd -----------------------------------------------------------------------------------
// A result in other sizes, no view to autograd: it may be changed in place.
Tensor in_sizes(const Tensor& t, at::IntArrayRef sizes) {
    at::AutoDispatchBelowADInplaceOrView below;
    return t.view(sizes);
}
OptTensor defined(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// A tangent of forward mode (a tensor has one whether or not it requires grad) would be dropped.
void no_tangent(const char* fn, const Tensor& t) {
    if (t._fw_grad(/*level=*/0).defined()) refuse(fn, "forward-mode differentiation is not available");
}
void no_tangent(const char* fn, const OptTensor& t) {
    if (t) no_tangent(fn, *t);
}

// The gradients are made by the kernels, without a graph of their own.  Under create_graph a gradient `g`
// is handed on with this node: differentiating it raises, where without the node the terms that it
// contributes to a second derivative would just be missing.
struct OnceFn : torch::autograd::Function<OnceFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& g, const Tensor& /* requires grad */, const std::string& fn) {
        ctx->saved_data["fn"] = fn;
        return g.variable_data();  // (ours alone, and no view: in-place changes of the gradient stay allowed)
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list&) {
        refuse(ctx->saved_data["fn"].toStringRef().c_str(), "second derivatives are not available");
    }
};
Tensor once(const char* fn, const Tensor& g) {
    if (!g.defined() || !at::GradMode::is_enabled()) return g;
    return OnceFn::apply(g, at::empty({0}, at::kFloat).requires_grad_(), std::string(fn));
}
// The same for a gradient whose memory is another one's too, the caller's or a second gradient: under create_graph a copy,
// as in-place changes of what OnceFn hands on raise no other tensor's version.
Tensor once_shared(const char* fn, const Tensor& g) {
    if (!g.defined() || !at::GradMode::is_enabled()) return g;
    return once(fn, g.detach().clone());
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& gamma, const OptTensor& beta,
                          double eps) {
        const NormOut n = layer_norm(x, gamma, beta, eps, std::nullopt, true);
        ctx->save_for_backward({x, gamma ? *gamma : Tensor(), n.mean, n.rstd});
        ctx->saved_data["params"] = (gamma && gamma->requires_grad()) || (beta && beta->requires_grad());
        ctx->saved_data["beta"] = beta ? static_cast<int64_t>(beta->scalar_type()) : static_cast<int64_t>(-1);
        return n.y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
        const auto saved = ctx->get_saved_variables();
        const NormGrad g = layer_norm_backward(dy[0].contiguous(), saved[0], saved[2], saved[3], defined(saved[1]),
                                               ctx->saved_data["params"].toBool());
        const int64_t bt = ctx->saved_data["beta"].toInt();
        Tensor db = g.dbeta;
        if (db.defined() && bt >= 0) db = db.to(static_cast<at::ScalarType>(bt));
        const char* fn = "layer_norm_autograd";
        return {once(fn, g.dx), saved[1].defined() ? once(fn, g.dgamma) : Tensor(), bt >= 0 ? once(fn, db) : Tensor(), Tensor()};
    }
};

// y = Q(x) Q(W)^T + b; dx = Q(dy) Q(W^T)^T, dW = Q(dy^T) Q(x^T)^T, db = sums of dy's columns.  The transposed
// operands of the backward products are made with the forward ones, from the same reads.
struct Fp8LinearFn : torch::autograd::Function<Fp8LinearFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b) {
        const bool dx = x.requires_grad(), dw = w.requires_grad(), db = b && b->requires_grad();
        const Quantised xq = fp8_quantise(x, false, dw, false), wq = fp8_quantise(w, true, dx, false);
        const Tensor none;
        ctx->save_for_backward({dw ? xq.qt->codes : none, dw ? xq.qt->scales : none, dx ? wq.qt->codes : none,
                                dx ? wq.qt->scales : none});
        ctx->saved_data["db"] = db;
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["types"] = std::vector<int64_t>{static_cast<int64_t>(x.scalar_type()), static_cast<int64_t>(w.scalar_type()),
                                                        b ? static_cast<int64_t>(b->scalar_type()) : 0};
        auto sizes = x.sizes().vec();
        sizes.back() = w.size(0);
        return in_sizes(fp8_gemm(xq.q.codes, xq.q.scales, false, wq.q.codes, wq.q.scales, true, b, 0, x.scalar_type(), std::nullopt), sizes);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto types = ctx->saved_data["types"].toIntVector();
        const bool need_dw = saved[0].defined(), need_dx = saved[2].defined(), need_db = ctx->saved_data["db"].toBool();
        const Tensor dy = grads[0].contiguous();
        // one read of dy makes the operands of both products and the bias gradient
        const Quantised q = fp8_quantise(dy, false, need_dw, need_db,
                                         need_db ? static_cast<at::ScalarType>(types[2]) : at::kFloat);
        Tensor dx, dw;
        if (need_dw)
            dw = fp8_gemm(q.qt->codes, q.qt->scales, false, saved[0], saved[1], false, std::nullopt, 0,
                          static_cast<at::ScalarType>(types[1]), std::nullopt);
        if (need_dx)
            dx = fp8_gemm(q.q.codes, q.q.scales, false, saved[2], saved[3], true, std::nullopt, 0,
                          static_cast<at::ScalarType>(types[0]), std::nullopt).view(ctx->saved_data["x"].toIntVector());
        const char* fn = "fp8_linear";
        return {once(fn, dx), once(fn, dw), once(fn, q.sums)};
    }
};

Tensor fp8_linear(const Tensor& x, const Tensor& w, const OptTensor& b) {
    const char* fn = "fp8_linear";
    type_of(fn, "x", x);
    type_of(fn, "weight", w);
    if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1))
        refuse(fn, "weight must be (N, " + (x.dim() ? std::to_string(x.size(-1)) : std::string("?")) + ")");
    same_device(fn, x, "weight", w);
    int t = 0;
    vector_of(fn, "bias", b, w.size(0), x, &t);
    no_tangent(fn, x), no_tangent(fn, w), no_tangent(fn, b);
    if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (b && b->requires_grad())))
        return Fp8LinearFn::apply(x, w, b);
    // no gradient is asked for: no transposed operands
    const Quantised xq = fp8_quantise(x, false, false, false), wq = fp8_quantise(w, true, false, false);
    auto sizes = x.sizes().vec();
    sizes.back() = w.size(0);
    return in_sizes(fp8_gemm(xq.q.codes, xq.q.scales, false, wq.q.codes, wq.q.scales, true, b, 0, x.scalar_type(), std::nullopt), sizes);
}

#include "nfx_torch_dense.h"

py::object or_none(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

}  // namespace

PYBIND11_MODULE(_nfx_torch, m) {
    m.def("layer_norm", [](const Tensor& x, const OptTensor& g, const OptTensor& b, double eps, const OptTensor& out, bool stats) {
        const NormOut n = layer_norm(x, g, b, eps, out, stats);
        return stats ? py::object(py::make_tuple(n.y, n.mean, n.rstd)) : py::cast(n.y);
    });
    m.def("layer_norm_fp8", &layer_norm_fp8);
    m.def("layer_norm_backward", [](const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd, const OptTensor& g,
                                    bool params) {
        const NormGrad n = layer_norm_backward(dy, x, mean, rstd, g, params);
        return py::make_tuple(n.dx, or_none(n.dgamma), or_none(n.dbeta));
    });
    m.def("fp8_quantise", [](const Tensor& x, bool tile, bool transposed, bool col_sums) {
        const Quantised q = fp8_quantise(x, tile, transposed, col_sums);
        return py::make_tuple(q.q.codes, q.q.scales, q.qt ? py::object(py::make_tuple(q.qt->codes, q.qt->scales)) : py::none(),
                              or_none(q.sums));
    });
    m.def("fp8_gemm", &fp8_gemm);
    m.def("fp8_linear", &fp8_linear);
    m.def("layer_norm_autograd", [](const Tensor& x, const OptTensor& g, const OptTensor& b, double eps) {
        const char* fn = "layer_norm_autograd";
        norm_of(fn, x, g, b);
        no_tangent(fn, x), no_tangent(fn, g), no_tangent(fn, b);
        const bool grad = x.requires_grad() || (g && g->requires_grad()) || (b && b->requires_grad());
        if (!grad || !at::GradMode::is_enabled()) return layer_norm(x, g, b, eps, std::nullopt, false).y;
        return Tensor(LayerNormFn::apply(x, g, b, eps));
    });
    dense_defs(m);
}
