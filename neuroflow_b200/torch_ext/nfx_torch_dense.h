// nfx_torch_dense.h -- the part of the torch front-end (nfx_torch.cpp, which includes it) for the operators of
// a pre-norm block in 16 bits: RMS norm with the residual's addition, the product with bias, activation and
// residual, the activation's gradient, and gradient clipping.
#pragma once

// ---- memory that a call reads and writes ---------------------------------------------------------
// Evenly strided rows of a tensor as bytes.
struct Span {
    uintptr_t at;
    int64_t rows, width, pitch;
};
Span span_of(const Tensor& t, const Rows& r) {
    const int64_t e = static_cast<int64_t>(t.element_size());
    return {reinterpret_cast<uintptr_t>(t.const_data_ptr()), r.cols > 0 ? r.rows : 0, r.cols * e, r.ld * e};
}
// Whether two of them may share a byte: rows side by side with one pitch do not (the columns of a wider
// matrix); anything else that reaches into the other's range is taken to.
bool may_share(const Span& a, const Span& b) {
    if (a.rows == 0 || b.rows == 0) return false;
    const auto end = [](const Span& s) { return s.at + static_cast<uintptr_t>((s.rows - 1) * s.pitch + s.width); };
    if (end(a) <= b.at || end(b) <= a.at) return false;
    if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch)) return true;
    const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    // where b's row starts within a's pitch
    const int64_t off = b.at >= a.at ? static_cast<int64_t>((b.at - a.at) % static_cast<uintptr_t>(pitch))
                                     : (pitch - static_cast<int64_t>((a.at - b.at) % static_cast<uintptr_t>(pitch))) % pitch;
    return !(off >= a.width && off + b.width <= pitch);
}
bool same_rows(const Span& a, const Span& b) { return a.at == b.at && a.rows == b.rows && a.width == b.width && (a.rows <= 1 || a.pitch == b.pitch); }

// `out` must not share memory with what is read, save for being the very rows of it where `same` allows that.
void apart(const char* fn, const char* name, const Tensor& out, const Rows& r, const char* other_name, const Tensor& other,
           const Rows& o, bool same) {
    const Span a = span_of(out, r), b = span_of(other, o);
    if (same && same_rows(a, b) && out.scalar_type() == other.scalar_type()) return;
    if (may_share(a, b)) refuse(fn, std::string(name) + " shares memory with " + other_name);
}

// A given output of this shape and type, on x's device.
Rows out_of(const char* fn, const char* name, const Tensor& out, at::IntArrayRef sizes, at::ScalarType type, const Tensor& x) {
    if (out.sizes() != sizes || out.scalar_type() != type || out.device() != x.device())
        refuse(fn, std::string(name) + " must have the result's shape, its type (" + c10::toString(type) + ") and x's device");
    if (out.requires_grad() && at::GradMode::is_enabled()) refuse(fn, std::string(name) + " must not be a tensor that requires grad");
    return rows_of(fn, name, out);
}

Tensor workspace(int64_t bytes, const Tensor& like) { return bytes > 0 ? empty({bytes}, at::kByte, like) : Tensor(); }
void* raw(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- RMS norm -------------------------------------------------------------------------------------
struct Rms {
    Rows x, res{}, sum{};
    int xt, ht, pt = NFX_F32;
    const void *g, *r = nullptr;
    Tensor h;  // x + residual, where there is one
    Tensor rstd;
};
Rms rms_of(const char* fn, const Tensor& x, const OptTensor& gamma, const OptTensor& residual, const OptTensor& sum_out) {
    Rms n;
    n.xt = n.ht = type_of(fn, "x", x);
    n.x = rows_of(fn, "x", x);
    if (n.x.cols < 1) refuse(fn, "the last dimension is empty");
    n.g = vector_of(fn, "gamma", gamma, n.x.cols, x, &n.pt);
    if (sum_out && !residual) refuse(fn, "sum_out is for the sum with a residual");
    if (residual) {
        n.ht = type_of(fn, "residual", *residual);
        same_device(fn, x, "residual", *residual);
        if (residual->sizes() != x.sizes()) refuse(fn, "residual must have x's shape");
        if (n.ht != n.xt && n.ht != NFX_F32) refuse(fn, "residual must have x's type or be float32");
        n.res = rows_of(fn, "residual", *residual);
        n.r = residual->const_data_ptr();
        if (sum_out) {
            n.sum = out_of(fn, "sum_out", *sum_out, x.sizes(), residual->scalar_type(), x);
            apart(fn, "sum_out", *sum_out, n.sum, "x", x, n.x, true);
            apart(fn, "sum_out", *sum_out, n.sum, "residual", *residual, n.res, true);
            if (gamma) apart(fn, "sum_out", *sum_out, n.sum, "gamma", *gamma, {1, n.x.cols, n.x.cols}, false);
        }
    }
    return n;
}
// the outputs that both forms have (allocated on x's device, which is current)
void rms_outputs(Rms& n, const Tensor& x, const OptTensor& residual, const OptTensor& sum_out, bool stats) {
    if (residual) {
        n.h = sum_out ? *sum_out : empty(x.sizes(), residual->scalar_type(), x);
        if (!sum_out) n.sum = {n.x.rows, n.x.cols, n.x.cols};
    }
    if (stats) n.rstd = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
}

struct RmsOut {
    Tensor y, h, rstd;
};
RmsOut rms_norm(const Tensor& x, const OptTensor& gamma, double eps, const OptTensor& residual, const OptTensor& out,
                const OptTensor& sum_out, bool stats) {
    const char* fn = "rms_norm";
    Rms n = rms_of(fn, x, gamma, residual, sum_out);
    Rows ry{n.x.rows, n.x.cols, n.x.cols};
    if (out) {
        ry = out_of(fn, "out", *out, x.sizes(), x.scalar_type(), x);
        apart(fn, "out", *out, ry, "x", x, n.x, true);
        if (residual) apart(fn, "out", *out, ry, "residual", *residual, n.res, true);
        if (sum_out) apart(fn, "out", *out, ry, "sum_out", *sum_out, n.sum, false);
        if (gamma) apart(fn, "out", *out, ry, "gamma", *gamma, {1, n.x.cols, n.x.cols}, false);
    }
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = out ? *out : empty(x.sizes(), x.scalar_type(), x);
    rms_outputs(n, x, residual, sum_out, stats);
    check(nfx_rms_norm(x.const_data_ptr(), n.xt, n.x.ld, n.r, n.ht, n.res.ld, n.g, n.pt, n.x.rows, n.x.cols, static_cast<float>(eps),
                       y.data_ptr(), ry.ld, raw(n.h), n.sum.ld, ptr(n.rstd), stream_of(x)));
    written(out), written(sum_out);
    return {y, n.h, n.rstd};
}

py::object rms_norm_fp8(const Tensor& x, const OptTensor& gamma, double eps, const OptTensor& residual, const OptTensor& sum_out,
                        bool stats) {
    Rms n = rms_of("rms_norm_fp8", x, gamma, residual, sum_out);
    c10::cuda::CUDAGuard guard(x.device());
    const Fp8 q(n.x.rows, n.x.cols, n.x.rows, x);
    rms_outputs(n, x, residual, sum_out, stats);
    check(nfx_rms_norm_fp8(x.const_data_ptr(), n.xt, n.x.ld, n.r, n.ht, n.res.ld, n.g, n.pt, n.x.rows, n.x.cols,
                           static_cast<float>(eps), q.data(), q.ld, q.scale(), 1, q.srows, raw(n.h), n.sum.ld, ptr(n.rstd),
                           stream_of(x)));
    written(sum_out);
    return py::make_tuple(q.codes, q.scales, n.h.defined() ? py::cast(n.h) : py::none(), n.rstd.defined() ? py::cast(n.rstd) : py::none());
}

struct RmsGrad {
    Tensor dx, dres, dgamma;
};
// dx of dy's type and dres of h's: one tensor where the types are equal; only those that are asked for.
RmsGrad rms_norm_backward(const Tensor& dy, const Tensor& h, const Tensor& rstd, const OptTensor& gamma, const OptTensor& dsum,
                          bool param_grads, bool need_dx = true, bool need_dres = true) {
    const char* fn = "rms_norm_backward";
    const int yt = type_of(fn, "dy", dy), ht = type_of(fn, "h", h);
    const Rows rh = rows_of(fn, "h", h);
    if (rh.cols < 1) refuse(fn, "the last dimension is empty");
    if (dy.sizes() != h.sizes()) refuse(fn, "dy must have h's shape");
    if (ht != yt && ht != NFX_F32) refuse(fn, "h must have dy's type or be float32");
    const Rows rdy = rows_of(fn, "dy", dy);
    same_device(fn, h, "dy", dy);
    int pt = NFX_F32;
    const void* g = vector_of(fn, "gamma", gamma, rh.cols, h, &pt);
    if (type_of(fn, "rstd", rstd) != NFX_F32 || rstd.numel() != rh.rows || !rstd.is_contiguous())
        refuse(fn, "rstd must be a contiguous float32 tensor of " + std::to_string(rh.rows));
    same_device(fn, h, "rstd", rstd);
    Rows rds{};
    if (dsum) {
        if (type_of(fn, "dsum", *dsum) != ht || dsum->sizes() != h.sizes()) refuse(fn, "dsum must have h's shape and type");
        same_device(fn, h, "dsum", *dsum);
        rds = rows_of(fn, "dsum", *dsum);
    }
    c10::cuda::CUDAGuard guard(h.device());
    const bool one = yt == ht;
    RmsGrad o;
    if (need_dx || (one && need_dres)) o.dx = empty(h.sizes(), dy.scalar_type(), h);
    if (!one && need_dres) o.dres = empty(h.sizes(), h.scalar_type(), h);
    Tensor ws;
    int64_t bytes = 0;
    if (param_grads) {
        o.dgamma = empty({rh.cols}, gamma ? gamma->scalar_type() : at::kFloat, h);
        bytes = nfx_rms_norm_backward_workspace(rh.rows, rh.cols);
        ws = workspace(bytes, h);
    }
    check(nfx_rms_norm_backward(dy.const_data_ptr(), yt, rdy.ld, h.const_data_ptr(), ht, rh.ld,
                                static_cast<const float*>(rstd.const_data_ptr()), g, pt, dsum ? dsum->const_data_ptr() : nullptr,
                                rds.ld, rh.rows, rh.cols, raw(o.dx), rh.cols, raw(o.dres), rh.cols, raw(o.dgamma), raw(ws), bytes,
                                stream_of(h)));
    if (one) o.dres = o.dx;
    return o;
}

// ---- product --------------------------------------------------------------------------------------
// A matrix whose rows or whose columns are contiguous.
struct Matrix {
    int64_t rows, cols, ld;
    int t;
    const void* p;
};
Matrix matrix_of(const char* fn, const char* name, const Tensor& m, at::ScalarType type) {
    if (!m.is_cuda()) refuse(fn, std::string(name) + " must be a CUDA tensor");
    if (m.scalar_type() != type) refuse(fn, std::string(name) + " must be " + c10::toString(type) + ", not " + c10::toString(m.scalar_type()));
    if (m.dim() != 2) refuse(fn, std::string(name) + " must have two dimensions");
    const int64_t r = m.size(0), c = m.size(1), sr = m.stride(0), sc = m.stride(1);
    const void* p = m.const_data_ptr();
    if (m.numel() == 0) return {r, c, c, 0, p};
    if ((c == 1 || sc == 1) && (r == 1 || sr >= c)) return {r, c, r == 1 ? c : sr, 0, p};
    if ((r == 1 || sr == 1) && (c == 1 || sc >= r)) return {r, c, c == 1 ? r : sc, 1, p};
    refuse(fn, "the rows or the columns of " + std::string(name) + " must be contiguous and must not overlap");
}
Rows rows_of(const Matrix& m) { return m.t ? Rows{m.cols, m.rows, m.ld} : Rows{m.rows, m.cols, m.ld}; }
at::ScalarType operand_type(const char* fn, const char* name, const Tensor& a) {
    if (!a.is_cuda()) refuse(fn, std::string(name) + " must be a CUDA tensor");
    if (a.scalar_type() != at::kBFloat16 && a.scalar_type() != at::kHalf)
        refuse(fn, std::string(name) + " must be bfloat16 or float16, not " + c10::toString(a.scalar_type()));
    return a.scalar_type();
}

struct Product {
    Tensor c, z;
};
Product gemm(const char* fn, const Tensor& at, const Tensor& bt, const OptTensor& bias, int64_t act, const OptTensor& residual,
             std::optional<at::ScalarType> out_dtype, const OptTensor& out, bool preact) {
    const at::ScalarType type = operand_type(fn, "a", at);
    const Matrix a = matrix_of(fn, "a", at, type), b = matrix_of(fn, "b", bt, type);
    if (a.cols != b.cols) refuse(fn, "a has " + std::to_string(a.cols) + " columns and b " + std::to_string(b.cols));
    same_device(fn, at, "b", bt);
    if (act < 0 || act > 2) refuse(fn, "act must be 0, 1 or 2");
    int bt_type = NFX_F32;
    const void* bp = vector_of(fn, "bias", bias, b.rows, at, &bt_type);
    const int64_t sizes[2] = {a.rows, b.rows};
    const at::ScalarType ct = out ? out->scalar_type() : (out_dtype ? *out_dtype : type);
    if (ct != type && ct != at::kFloat) refuse(fn, std::string("the result must be of the operands' type or float32, not ") + c10::toString(ct));
    if (out && out_dtype && *out_dtype != ct) refuse(fn, "out is not of out_dtype");
    Rows rc{a.rows, b.rows, b.rows}, rr{};
    const void* rp = nullptr;
    if (residual) {
        if (residual->sizes() != at::IntArrayRef(sizes, 2) || type_of(fn, "residual", *residual) != type_of(ct))
            refuse(fn, "residual must have the result's shape and type");
        same_device(fn, at, "residual", *residual);
        rr = rows_of(fn, "residual", *residual);
        rp = residual->const_data_ptr();
    }
    if (out) {
        if (!out->is_cuda()) refuse(fn, "out must be a CUDA tensor");
        rc = out_of(fn, "out", *out, at::IntArrayRef(sizes, 2), ct, at);
        apart(fn, "out", *out, rc, "a", at, rows_of(a), false);
        apart(fn, "out", *out, rc, "b", bt, rows_of(b), false);
        if (bias) apart(fn, "out", *out, rc, "bias", *bias, {1, b.rows, b.rows}, false);
        if (residual) apart(fn, "out", *out, rc, "residual", *residual, rr, true);
    }
    c10::cuda::CUDAGuard guard(at.device());
    Product o;
    o.c = out ? *out : empty(at::IntArrayRef(sizes, 2), ct, at);
    if (preact) o.z = empty(at::IntArrayRef(sizes, 2), ct, at);
    const int64_t bytes = nfx_gemm_workspace(a.p, a.ld, a.t, b.p, b.ld, b.t, a.rows, b.rows, a.cols);
    const Tensor ws = workspace(bytes, at);
    check(nfx_gemm(a.p, a.ld, a.t, b.p, b.ld, b.t, type_of(type), a.rows, b.rows, a.cols, bp, bt_type, static_cast<int>(act), rp, rr.ld,
                   o.c.data_ptr(), type_of(ct), rc.ld, raw(o.z), b.rows, raw(ws), bytes, stream_of(at)));
    written(out);
    return o;
}

Matrix transposed(const Matrix& m) { return {m.cols, m.rows, m.ld, 1 - m.t, m.p}; }
// a b^T of `type` as a tensor of `sizes`, the product's elements in order.
Tensor plain_product(const Matrix& a, const Matrix& b, at::ScalarType type, at::IntArrayRef sizes, const Tensor& like) {
    c10::cuda::CUDAGuard guard(like.device());
    const Tensor c = empty(sizes, type, like);
    const int64_t bytes = nfx_gemm_workspace(a.p, a.ld, a.t, b.p, b.ld, b.t, a.rows, b.rows, a.cols);
    const Tensor ws = workspace(bytes, like);
    check(nfx_gemm(a.p, a.ld, a.t, b.p, b.ld, b.t, type_of(type), a.rows, b.rows, a.cols, nullptr, NFX_F32, 0, nullptr, 0, c.data_ptr(), type_of(type),
                   b.rows, nullptr, b.rows, raw(ws), bytes, stream_of(like)));
    return c;
}

struct ActGrad {
    Tensor dz, db;
};
// dz is not made where it would be dy (no activation).
ActGrad act_backward(const char* fn, const Tensor& dy, const OptTensor& z, int64_t act, bool need_dz, std::optional<at::ScalarType> db_type) {
    const int t = type_of(fn, "dy", dy);
    const Rows r = rows_of(fn, "dy", dy);
    if (act < 0 || act > 2) refuse(fn, "act must be 0, 1 or 2");
    Rows rz{};
    const void* zp = nullptr;
    if (act) {
        if (!z) refuse(fn, "z is needed with an activation");
        if (type_of(fn, "z", *z) != t || z->sizes() != dy.sizes()) refuse(fn, "z must have dy's shape and type");
        same_device(fn, dy, "z", *z);
        rz = rows_of(fn, "z", *z);
        zp = z->const_data_ptr();
    }
    c10::cuda::CUDAGuard guard(dy.device());
    ActGrad o;
    if (need_dz) o.dz = act ? empty(dy.sizes(), dy.scalar_type(), dy) : dy;
    Tensor ws;
    int64_t bytes = 0;
    if (db_type) {
        o.db = empty({r.cols}, *db_type, dy);
        bytes = nfx_act_backward_workspace(r.rows, r.cols);
        ws = workspace(bytes, dy);
    }
    if ((need_dz && act) || db_type)
        check(nfx_act_backward(dy.const_data_ptr(), r.ld, zp, rz.ld, t, static_cast<int>(act), r.rows, r.cols,
                               need_dz && act ? o.dz.data_ptr() : nullptr, r.cols, raw(o.db), db_type ? type_of(*db_type) : static_cast<int>(NFX_F32),
                               raw(ws), bytes, stream_of(dy)));
    return o;
}

// ---- gradient norm --------------------------------------------------------------------------------
// A Python list of tensors, which are read where they are: a list of hundreds is looked at tensor by tensor while
// nothing else of the call takes as long.
class TensorList {
    py::list held_;
    std::vector<const Tensor*> t_;

public:
    TensorList(const char* what, py::list list) : held_(std::move(list)) {
        const Py_ssize_t n = PyList_GET_SIZE(held_.ptr());
        t_.reserve(static_cast<size_t>(n));
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* const o = PyList_GET_ITEM(held_.ptr(), i);
            if (!THPVariable_CheckExact(o) && !THPVariable_Check(o)) throw py::type_error(std::string(what) + " must be tensors");
            t_.push_back(&THPVariable_Unpack(o));
        }
    }
    size_t size() const { return t_.size(); }
    const Tensor& operator[](size_t i) const { return *t_[i]; }
};
struct GradList {
    std::vector<const void*> src;
    std::vector<void*> dst;
    std::vector<int64_t> n;
    std::vector<int> types, dst_types;
};
int64_t bytes_of(int type) { return type == NFX_F32 ? 4 : 2; }
void no_overlap(const char* fn, const GradList& l, bool out) {
    struct Part {
        uintptr_t at, end;
        bool write;
    };
    std::vector<Part> p;
    p.reserve(l.n.size() * 2);
    for (size_t i = 0; i < l.n.size(); ++i) {
        if (l.n[i] == 0) continue;
        const uintptr_t s = reinterpret_cast<uintptr_t>(l.src[i]);
        const uintptr_t d = out ? reinterpret_cast<uintptr_t>(l.dst[i]) : s;
        const int dt = out ? l.dst_types[i] : l.types[i];
        if (d != s || dt != l.types[i]) p.push_back({s, s + static_cast<uintptr_t>(l.n[i] * bytes_of(l.types[i])), false});
        p.push_back({d, d + static_cast<uintptr_t>(l.n[i] * bytes_of(dt)), true});
    }
    const auto before = [](const Part& a, const Part& b) { return a.at < b.at; };
    if (!std::is_sorted(p.begin(), p.end(), before)) std::sort(p.begin(), p.end(), before);
    uintptr_t read_end = 0, write_end = 0;
    for (const Part& q : p) {
        if (q.at < write_end || (q.write && q.at < read_end)) refuse(fn, out ? "an out shares memory with another tensor" : "two of the gradients share memory");
        (q.write ? write_end : read_end) = std::max(q.write ? write_end : read_end, q.end);
    }
}
GradList grads_of(const char* fn, const TensorList& g, const TensorList* out) {
    if (g.size() == 0) refuse(fn, "there are no gradients");
    if (out && out->size() != g.size()) refuse(fn, "out must have a tensor for each gradient");
    GradList l;
    l.src.reserve(g.size()), l.n.reserve(g.size()), l.types.reserve(g.size());
    if (out) l.dst.reserve(g.size()), l.dst_types.reserve(g.size());
    for (size_t i = 0; i < g.size(); ++i) {
        const Tensor& t = g[i];
        if (!t.defined() || t.layout() != at::kStrided) refuse(fn, "a gradient must be a dense tensor");
        l.types.push_back(type_of(fn, "a gradient", t));
        same_device(fn, g[0], "a gradient", t);
        if (!t.is_contiguous() && !t.is_non_overlapping_and_dense()) refuse(fn, "a gradient must be contiguous, or a permutation of a contiguous tensor");
        l.src.push_back(t.const_data_ptr());
        l.n.push_back(t.numel());
        if (!out) continue;
        const Tensor& o = (*out)[i];
        if (!o.defined() || o.layout() != at::kStrided) refuse(fn, "an out must be a dense tensor");
        l.dst_types.push_back(type_of(fn, "an out", o));
        same_device(fn, g[0], "an out", o);
        if (o.sizes() != t.sizes() || !((o.is_contiguous() && t.is_contiguous()) || (o.strides() == t.strides())))
            refuse(fn, "an out must have its gradient's shape and order of dimensions");
        l.dst.push_back(o.data_ptr());
    }
    return l;
}

Tensor grad_norm(py::list grads) {
    const char* fn = "grad_norm";
    const TensorList g("gradients", std::move(grads));
    const GradList l = grads_of(fn, g, nullptr);
    c10::cuda::CUDAGuard guard(g[0].device());
    const Tensor norm = empty({}, at::kFloat, g[0]);
    const int64_t bytes = nfx_grad_norm_workspace(static_cast<int64_t>(g.size()));
    const Tensor ws = workspace(bytes, g[0]);
    check(nfx_grad_norm(l.src.data(), l.n.data(), l.types.data(), static_cast<int64_t>(g.size()), ptr(norm), raw(ws), bytes, stream_of(g[0])));
    return norm;
}

Tensor clip_grad_norm(py::list grads, double max_norm, double eps, std::optional<py::list> outs) {
    const char* fn = "clip_grad_norm";
    const bool out = outs.has_value();
    const TensorList g("gradients", std::move(grads)), o("out", out ? std::move(*outs) : py::list());
    const TensorList& to = out ? o : g;
    if (!(max_norm >= 0)) refuse(fn, "max_norm must be >= 0");
    if (!(eps >= 0) || std::isinf(eps)) refuse(fn, "eps must be >= 0 and finite");
    const GradList l = grads_of(fn, g, out ? &o : nullptr);
    if (at::GradMode::is_enabled())
        for (size_t i = 0; i < to.size(); ++i)
            if (to[i].requires_grad()) refuse(fn, "a tensor that is written must not require grad");
    no_overlap(fn, l, out);
    c10::cuda::CUDAGuard guard(g[0].device());
    const Tensor norm = empty({}, at::kFloat, g[0]);
    const int64_t bytes = nfx_grad_norm_workspace(static_cast<int64_t>(g.size()));
    const Tensor ws = workspace(bytes, g[0]);
    check(nfx_clip_grad_norm(l.src.data(), l.n.data(), l.types.data(), out ? l.dst.data() : nullptr, out ? l.dst_types.data() : nullptr,
                             static_cast<int64_t>(g.size()), max_norm, eps, ptr(norm), raw(ws), bytes, stream_of(g[0])));
    for (size_t i = 0; i < to.size(); ++i)
        if (!to[i].is_inference()) to[i].unsafeGetTensorImpl()->bump_version();
    return norm;
}

// ---- autograd -------------------------------------------------------------------------------------
struct RmsNormFn : torch::autograd::Function<RmsNormFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& gamma, double eps,
                                                  const OptTensor& residual) {
        const RmsOut n = rms_norm(x, gamma, eps, residual, std::nullopt, std::nullopt, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual ? n.h : x, gamma ? *gamma : Tensor(), n.rstd});
        ctx->saved_data["xtype"] = static_cast<int64_t>(x.scalar_type());
        ctx->saved_data["needs"] = (x.requires_grad() ? 1 : 0) | (gamma && gamma->requires_grad() ? 2 : 0) |
                                   (residual && residual->requires_grad() ? 4 : 0);
        if (residual) return {n.y, n.h};
        return {n.y};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const char* fn = "rms_norm_autograd";
        const auto saved = ctx->get_saved_variables();
        const int64_t needs = ctx->saved_data["needs"].toInt();
        const Tensor dy = grads[0], ds = grads.size() > 1 ? grads[1] : Tensor();
        if (!dy.defined()) {  // only the sum is used: its gradient is that of both terms
            const auto as = [&](bool need, at::ScalarType t) { return need && ds.defined() ? once_shared(fn, ds.to(t)) : Tensor(); };
            return {as(needs & 1, static_cast<at::ScalarType>(ctx->saved_data["xtype"].toInt())), Tensor(), Tensor(),
                    as(needs & 4, ds.defined() ? ds.scalar_type() : at::kFloat)};
        }
        RmsGrad g = rms_norm_backward(dy.contiguous(), saved[0], saved[2], defined(saved[1]),
                                      ds.defined() ? OptTensor(ds.contiguous()) : std::nullopt, (needs & 2) != 0, (needs & 1) != 0,
                                      (needs & 4) != 0);
        return {needs & 1 ? once(fn, g.dx) : Tensor(), needs & 2 ? once(fn, g.dgamma) : Tensor(), Tensor(),
                needs & 4 ? ((needs & 1) && g.dres.is_same(g.dx) ? once_shared(fn, g.dres) : once(fn, g.dres)) : Tensor()};
    }
};

// y = act(x W^T + b) + R;  dz = dy act'(z), dx = dz W, dW = dz^T x, db = column sums of dz, dR = dy.  dz is rounded to
// x's type for the tensor cores.  z is kept in that type too, as fp32 would take twice the memory and traffic: half a
// step of z moves a GELU's dz by up to a third of it times |dy|, which is more than dz's own rounding where act' is small
// (2.5 times as much at z = -2).  The gradients of 4095x2048x8192 bf16 are 2.39e-3 of their norm off the 64-bit ones, with z in
// fp32 2.34e-3, with dz in fp32 1.73e-3; rounding the results alone gives 1.66e-3.
struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, int64_t act,
                          const OptTensor& residual, const Tensor& x2) {
        const OptTensor r2 = residual ? OptTensor(residual->reshape({x2.size(0), w.size(0)})) : std::nullopt;
        const bool grad_z = x.requires_grad() || w.requires_grad() || (b && b->requires_grad());
        const Product p = gemm("linear", x2, w, b, act, r2, std::nullopt, std::nullopt, act != 0 && grad_z);
        ctx->save_for_backward({w.requires_grad() ? x : Tensor(), x.requires_grad() ? w : Tensor(), p.z});
        // which gradients are wanted, the activation and the bias' type
        const int64_t needs = (x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0) | (b && b->requires_grad() ? 4 : 0) |
                              (residual && residual->requires_grad() ? 8 : 0);
        ctx->saved_data["what"] = needs | act << 4 | static_cast<int64_t>(b ? b->scalar_type() : at::kFloat) << 8;
        if (x.dim() == 2) return p.c;
        auto sizes = x.sizes().vec();
        sizes.back() = w.size(0);
        return in_sizes(p.c, sizes);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const char* fn = "linear";
        const auto saved = ctx->get_saved_variables();
        const int64_t what = ctx->saved_data["what"].toInt(), needs = what & 15, act = what >> 4 & 15;
        const Tensor dy = grads[0].contiguous();
        const at::ScalarType type = dy.scalar_type();
        int64_t rows = 1;
        for (int64_t i = 0; i + 1 < dy.dim(); ++i) rows *= dy.size(i);
        const auto flat = [&](const Tensor& t) { return t.dim() == 2 ? t : t.reshape({rows, t.size(-1)}); };
        Tensor dx, dw, db;
        if (needs & 7) {
            const ActGrad g = act_backward(fn, flat(dy), defined(saved[2]), act, (needs & 3) != 0,
                                           needs & 4 ? std::optional<at::ScalarType>(static_cast<at::ScalarType>(what >> 8)) : std::nullopt);
            db = g.db;
            if (needs & 2) {
                const Tensor x = flat(saved[0]);
                const int64_t sizes[2] = {dy.size(-1), x.size(1)};
                dw = plain_product(transposed(matrix_of(fn, "dy", g.dz, type)), transposed(matrix_of(fn, "x", x, type)), type, sizes, dy);
            }
            if (needs & 1) {
                auto sizes = dy.sizes().vec();
                sizes.back() = saved[1].size(1);
                dx = plain_product(matrix_of(fn, "dy", g.dz, type), transposed(matrix_of(fn, "weight", saved[1], type)), type, sizes, dy);
            }
        }
        return {once(fn, dx), once(fn, dw), once(fn, db), Tensor(), needs & 8 ? once_shared(fn, grads[0]) : Tensor(), Tensor()};
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const OptTensor& b, int64_t act, const OptTensor& residual) {
    const char* fn = "linear";
    const at::ScalarType type = operand_type(fn, "x", x);
    if (operand_type(fn, "weight", w) != type) refuse(fn, "weight must have x's type");
    if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1))
        refuse(fn, "weight must be (N, " + (x.dim() ? std::to_string(x.size(-1)) : std::string("?")) + ")");
    same_device(fn, x, "weight", w);
    auto sizes = x.sizes().vec();
    sizes.back() = w.size(0);
    if (residual && (residual->sizes() != at::IntArrayRef(sizes) || residual->scalar_type() != type))
        refuse(fn, "residual must have the result's shape and x's type");
    no_tangent(fn, x), no_tangent(fn, w), no_tangent(fn, b), no_tangent(fn, residual);
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) rows *= sizes[i];
    const auto flat = [&](const Tensor& t, int64_t cols) {
        at::AutoDispatchBelowADInplaceOrView below;
        return t.dim() == 2 ? t : t.reshape({rows, cols});
    };
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || w.requires_grad() || (b && b->requires_grad()) || (residual && residual->requires_grad())))
        return LinearFn::apply(x, w, b, act, residual, flat(x, w.size(1)));
    const OptTensor r2 = residual ? OptTensor(flat(*residual, w.size(0))) : std::nullopt;
    return in_sizes(gemm(fn, flat(x, w.size(1)), w, b, act, r2, std::nullopt, std::nullopt, false).c, sizes);
}

void dense_defs(py::module_& m) {
    m.def("rms_norm", [](const Tensor& x, const OptTensor& g, double eps, const OptTensor& res, const OptTensor& out,
                         const OptTensor& sum_out, bool stats) -> py::object {
        const RmsOut n = rms_norm(x, g, eps, res, out, sum_out, stats);
        if (res) return stats ? py::make_tuple(n.y, n.h, n.rstd) : py::make_tuple(n.y, n.h);
        return stats ? py::object(py::make_tuple(n.y, n.rstd)) : py::cast(n.y);
    });
    m.def("rms_norm_fp8", &rms_norm_fp8);
    m.def("rms_norm_backward", [](const Tensor& dy, const Tensor& h, const Tensor& rstd, const OptTensor& g, const OptTensor& dsum, bool params) {
        const RmsGrad n = rms_norm_backward(dy, h, rstd, g, dsum, params);
        return py::make_tuple(n.dx, n.dres, n.dgamma.defined() ? py::cast(n.dgamma) : py::none());
    });
    m.def("gemm", [](const Tensor& a, const Tensor& b, const OptTensor& bias, int64_t act, const OptTensor& res,
                     std::optional<at::ScalarType> out_dtype, const OptTensor& out, bool preact) -> py::object {
        const Product p = gemm("gemm", a, b, bias, act, res, out_dtype, out, preact);
        return preact ? py::object(py::make_tuple(p.c, p.z)) : py::cast(p.c);
    });
    m.def("act_backward", [](const Tensor& dy, const OptTensor& z, int64_t act, std::optional<at::ScalarType> db_type) {
        const ActGrad g = act_backward("act_backward", dy, z, act, true, db_type);
        return py::make_tuple(g.dz, g.db.defined() ? py::cast(g.db) : py::none());
    });
    m.def("grad_norm", &grad_norm);
    m.def("clip_grad_norm", &clip_grad_norm);
    m.def("linear", &linear);
    m.def("rms_norm_autograd", [](const Tensor& x, const OptTensor& g, double eps, const OptTensor& res) -> py::object {
        const char* fn = "rms_norm_autograd";
        rms_of(fn, x, g, res, std::nullopt);
        no_tangent(fn, x), no_tangent(fn, g), no_tangent(fn, res);
        const bool grad = x.requires_grad() || (g && g->requires_grad()) || (res && res->requires_grad());
        if (!grad || !at::GradMode::is_enabled()) {
            const RmsOut n = rms_norm(x, g, eps, res, std::nullopt, std::nullopt, false);
            return res ? py::object(py::make_tuple(n.y, n.h)) : py::cast(n.y);
        }
        const auto o = RmsNormFn::apply(x, g, eps, res);
        return res ? py::object(py::make_tuple(o[0], o[1])) : py::cast(o[0]);
    });
}
