// nfx_torch.cpp -- the torch front-end of the transformer-layer operators of libnfx.so (layer norm, FP8
// block quantiser, FP8 block-scaled product): checks of the tensors, allocation of the outputs on the
// current stream, and the C-ABI call, in compiled code because a call on one token takes the GPU a few
// microseconds and the same steps in Python ten or more.  neuroflow_b200/ops.py is the public face.
//
// Refused arguments raise neuroflow_b200._nfx.NfxError with status 1 (InvalidArg) before anything is
// launched; errors of the C-ABI raise it with theirs.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>

#include "nfx.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kGroup = 128;

[[noreturn]] void raise(int code, const std::string& msg) {
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
    py::tuple both() const { return py::make_tuple(codes, scales); }
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

py::object layer_norm(const Tensor& x, const OptTensor& gamma, const OptTensor& beta, double eps, const OptTensor& out, bool stats) {
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
    } else {
        y = empty(x.sizes(), x.scalar_type(), x);
    }
    std::pair<Tensor, Tensor> st;
    if (stats) st = stats_of(x);
    check(nfx_layer_norm(x.const_data_ptr(), n.xt, n.x.ld, n.g, n.b, n.pt, n.x.rows, n.x.cols, static_cast<float>(eps),
                         y.data_ptr(), ldy, ptr(st.first), ptr(st.second), stream_of(x)));
    if (!stats) return py::cast(y);
    return py::make_tuple(y, st.first, st.second);
}

py::object layer_norm_fp8(const Tensor& x, const OptTensor& gamma, const OptTensor& beta, double eps, bool stats) {
    const Norm n = norm_of("layer_norm_fp8", x, gamma, beta);
    c10::cuda::CUDAGuard guard(x.device());
    const Fp8 q(n.x.rows, n.x.cols, n.x.rows, x);
    std::pair<Tensor, Tensor> st;
    if (stats) st = stats_of(x);
    check(nfx_layer_norm_fp8(x.const_data_ptr(), n.xt, n.x.ld, n.g, n.b, n.pt, n.x.rows, n.x.cols, static_cast<float>(eps),
                             q.data(), q.ld, q.scale(), 1, q.srows, ptr(st.first), ptr(st.second), stream_of(x)));
    if (!stats) return q.both();
    return py::make_tuple(q.codes, q.scales, st.first, st.second);
}

py::tuple layer_norm_backward(const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd, const OptTensor& gamma,
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
    if (!param_grads) return py::make_tuple(dx, py::none(), py::none());
    return py::make_tuple(dx, dg, db);
}

py::tuple fp8_quantise(const Tensor& x, bool tile, bool transposed, bool col_sums) {
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
        sums = empty({r.cols}, at::kFloat, x);
        bytes = nfx_fp8_quantise_workspace(r.rows, r.cols);
        ws = empty({bytes}, at::kByte, x);
    }
    check(nfx_fp8_quantise(x.const_data_ptr(), xt, r.ld, r.rows, r.cols, tile, q.data(), q.ld, q.scale(), 1, q.srows,
                           qt ? qt->data() : nullptr, qt ? qt->ld : 0, qt ? qt->scale() : nullptr, 1, qt ? qt->srows : 0, ptr(sums),
                           col_sums ? ws.data_ptr() : nullptr, bytes, stream_of(x)));
    return py::make_tuple(q.codes, q.scales, qt ? py::object(qt->both()) : py::none(), col_sums ? py::cast(sums) : py::none());
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
    } else if (type_of(out_dtype) < 0) {
        refuse(fn, std::string("out_dtype must be float32, bfloat16 or float16, not ") + c10::toString(out_dtype));
    }
    c10::cuda::CUDAGuard guard(ac.device());
    if (!out) c = empty({a.rows, b.rows}, out_dtype, ac);
    check(nfx_fp8_gemm(a.codes, a.ld, a.scales, a.srs, a.sbs, a_tile, b.codes, b.ld, b.scales, b.srs, b.sbs, b_tile, a.rows, b.rows,
                       a.k, bp, bt, static_cast<int>(act), c.data_ptr(), type_of(c.scalar_type()), ldc, stream_of(ac)));
    return c;
}

}  // namespace

PYBIND11_MODULE(_nfx_torch, m) {
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_fp8", &layer_norm_fp8);
    m.def("layer_norm_backward", &layer_norm_backward);
    m.def("fp8_quantise", &fp8_quantise);
    m.def("fp8_gemm", &fp8_gemm);
}
