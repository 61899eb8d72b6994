"""RMS norm with the residual's addition (neuroflow_b200.ops.rms_norm* / nfx_rms_norm*) against its formula in
64 bits.

Tolerances.  eps = 2^-24 is the fp32 unit roundoff.  A row's sums are formed by threads that add at most
d / 32 elements one after another and then join in a tree or over warps, so with n = d / 32 + 48 a sum of
terms t is off by at most n eps sum |t| (a sum of squares by n eps of itself).
  h:      the fp32 sum of two numbers rounded once more to h's type: the same bits as torch's
  rstd:   half the sum's relative error, and four roundings: (n / 2 + 4) eps
  y:      two products on top: |y| (n / 2 + 7) eps, and half an ulp of the output type
  dh:     m = mean(a xh) is off by n eps mean|a xh|; a, xh, m xh, their difference, the product with rstd and the
          sum with dsum are rounded: r |xh| n eps mean|a xh| + 4 r eps (|a| + |xh m|) + 2 eps (|dh| + |dsum|),
          and half an ulp of the output type
  dgamma: rows' terms in any order: (rows + 4) eps sum |dy xh|, and half an ulp
"""
import pytest

pytestmark = pytest.mark.gpu
EPS32 = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half a step, relative
EPS = 1e-5
WIDTHS = [1, 2, 3, 31, 64, 66, 127, 128, 129, 256, 511, 514, 771, 1024, 1030, 1032, 2048, 2050, 4096, 4098, 5000, 8192, 9998,
          16384, 20001]
# x, residual (None: no residual), gamma
TYPES = [("float32", "float32", "float32"), ("bfloat16", "bfloat16", "bfloat16"), ("bfloat16", "float32", "float32"),
         ("float16", None, "float32"), ("float16", "float32", "float16"), ("float16", "float16", "float32"),
         ("bfloat16", None, None), ("float32", None, "bfloat16")]


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _tiny(dtype):
    return 2.0 ** -25 if dtype == "float16" else 1e-38


def _case(rows, d, x, h, g, seed, grad=False):
    torch, _ = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    dt = lambda n: getattr(torch, n)
    X = (rnd(rows, d) * torch.exp(0.5 * rnd(1, d)) + 0.2).to(dt(x))
    R = None if h is None else (2 * rnd(rows, d)).to(dt(h))
    G = None if g is None else (1 + 0.2 * rnd(d)).to(dt(g))
    if not grad:
        return X, R, G
    return X, R, G, (0.1 * rnd(rows, d)).to(dt(x)), None if h is None else (0.1 * rnd(rows, d)).to(dt(h))


def _plain(x, r, g, eps=EPS):
    """(y in 64 bits, h, rstd in 64 bits)"""
    h = x if r is None else (x.float() + r.float()).to(r.dtype)
    v = h.double()
    rstd = 1 / (v.square().mean(1) + eps).sqrt()
    y = v * rstd[:, None]
    return (y if g is None else y * g.double()), h, rstd


def _check_forward(y, h, rstd, x, r, g, eps=EPS):
    torch, _ = _torch()
    want, hw, rw = _plain(x, r, g, eps)
    n = x.shape[1] / 32 + 48
    if r is not None:
        assert h.dtype == r.dtype and torch.equal(h, hw)
    assert ((rstd.double() / rw - 1).abs() <= (n / 2 + 4) * EPS32).all()
    if y is not None:
        name = str(y.dtype)[6:]
        tol = want.abs() * ((n / 2 + 7) * EPS32 + HALF[name] * (1 + 1e-3)) + _tiny(name)
        assert y.dtype == x.dtype and ((y.double() - want).abs() <= tol).all()


def _grad_want(dy, h, rstd, g, ds):
    """(dh, its tolerance without the output's rounding, dgamma, sum |dy xh|)"""
    d = h.shape[1]
    n = d / 32 + 48
    D, xh = dy.double(), h.double() * rstd.double()[:, None]
    a = D if g is None else D * g.double()
    r = rstd.double()[:, None]
    m = (a * xh).mean(1, keepdim=True)
    dh = r * (a - xh * m)
    tol = r * xh.abs() * n * EPS32 * (a * xh).abs().mean(1, keepdim=True) + 4 * r * EPS32 * (a.abs() + (xh * m).abs())
    if ds is not None:
        dh = dh + ds.double()
        tol = tol + 2 * EPS32 * ds.double().abs()
    return dh, tol + 2 * EPS32 * dh.abs(), (D * xh).sum(0), (D * xh).abs().sum(0)


def _check_grad(dx, dres, dg, dy, h, rstd, g, ds):
    torch, _ = _torch()
    dh, tol, wg, mag = _grad_want(dy, h, rstd, g, ds)
    for got, like in ((dx, dy), (dres, h)):
        if got is None:
            continue
        name = str(got.dtype)[6:]
        assert got.dtype == like.dtype
        assert ((got.double() - dh).abs() <= tol + HALF[name] * (dh.abs() + tol) + _tiny(name)).all()
    if dg is not None:
        name = str(dg.dtype)[6:]
        t = (h.shape[0] + 4) * EPS32 * mag
        assert ((dg.double() - wg).abs() <= t + HALF[name] * (wg.abs() + t) + _tiny(name)).all()


@pytest.mark.parametrize("x,h,g", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_forward(d, x, h, g):
    torch, ops = _torch()
    for rows in (1, 3, 130):
        X, R, G = _case(rows, d, x, h, g, d + rows)
        got = ops.rms_norm(X, G, EPS, residual=R, stats=True)
        _check_forward(got[0], got[1], got[-1], X, R, G)
        again = ops.rms_norm(X, G, EPS, residual=R)
        assert torch.equal(again if R is None else again[0], got[0])


@pytest.mark.parametrize("x,h,g", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_backward(d, x, h, g):
    torch, ops = _torch()
    for rows in (1, 5, 133):
        X, R, G, dy, ds = _case(rows, d, x, h, g, d + rows, grad=True)
        _, hs, rstd = _plain(X, R, G)
        rstd = rstd.float()
        dx, dres, dg = ops.rms_norm_backward(dy, hs, rstd, G, dsum=ds)
        _check_grad(dx, dres, dg, dy, hs, rstd, G, ds)
        assert (dres is dx) == (hs.dtype == dy.dtype)
        only = ops.rms_norm_backward(dy, hs, rstd, G, dsum=ds, param_grads=False)
        assert torch.equal(only[0], dx) and only[2] is None
        assert all(torch.equal(p, q) for p, q in zip(ops.rms_norm_backward(dy, hs, rstd, G, dsum=ds), (dx, dres, dg)))


def test_many_rows():
    """More rows than blocks that walk over them."""
    torch, ops = _torch()
    for rows, d, x, h in ((70001, 64, "bfloat16", "bfloat16"), (9001, 1031, "float16", "float16"), (5000, 771, "float32", None),
                          (4103, 4096, "bfloat16", "float32")):
        X, R, G, dy, ds = _case(rows, d, x, h, "float32", rows, grad=True)
        got = ops.rms_norm(X, G, EPS, residual=R, stats=True)
        _check_forward(got[0], got[1], got[-1], X, R, G)
        hs = X if R is None else got[1]
        _check_grad(*ops.rms_norm_backward(dy, hs, got[-1], G, dsum=ds), dy, hs, got[-1], G, ds)


@pytest.mark.parametrize("x,h,g", TYPES[:6])
@pytest.mark.parametrize("d", [1, 31, 127, 128, 130, 500, 1031, 2048, 4096, 4102, 9998, 16384, 20001])
def test_fp8_form(d, x, h, g):
    """The codes and scales that fp8_quantise makes of y where y is in fp32, up to y's own rounding: a scale by
    that of its group's largest element, a value by an E4M3 half step (2^-4 of it, 2^-10 of a scale below the
    normal numbers, 2^-9 in the band that the encoder holds at the largest subnormal one) and y's."""
    torch, ops = _torch()
    for rows in (1, 70):
        X, R, G = _case(rows, d, x, h, g, 3 * d + rows)
        got = ops.rms_norm_fp8(X, G, EPS, residual=R, stats=True)
        _check_forward(None, got[1], got[-1], X, R, G)
        want, _, _ = _plain(X, R, G)
        n = d / 32 + 48
        err = (n / 2 + 7) * EPS32
        q = got[0]
        pad = torch.nn.functional.pad(want, (0, -d % 128)).view(rows, -1, 128)
        s = torch.clamp_min(pad.abs().amax(2) / 448, 2.0 ** -126)
        assert q.scales.shape == s.shape and ((q.scales.double() / s - 1).abs() <= err + 3 * EPS32).all()
        off = (q.dequantise().double() - want).abs()
        unit = q.scales.double().repeat_interleave(128, 1)[:, :d]
        assert (off <= want.abs() * (2.0 ** -4 + err + 4 * EPS32) + unit * 2.0 ** -9 * (1 + 1e-3)).all()
        # most codes are the nearest ones: those that a rounding of y moves over a boundary are few
        y32 = want.float()
        w = ops.fp8_quantise(y32)
        differ = (w.codes.view(torch.uint8) != q.codes.view(torch.uint8)).float().mean()
        assert differ <= 0.002 + 2 / (rows * d)


@pytest.mark.parametrize("x,h", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", None)])
@pytest.mark.parametrize("d,pitch,shift", [(256, 300, 0), (256, 256, 1), (1000, 1008, 8), (130, 133, 3), (4096, 4104, 2), (2047, 2047, 0),
                                           (1031, 1031, 5)])
def test_strides_and_alignment(d, pitch, shift, x, h):
    """Rows that start anywhere, in each tensor on its own; what lies between the rows is not written."""
    torch, ops = _torch()
    rows = 37
    X, R, G, dy, ds = _case(rows, d, x, h, "float32", 7, grad=True)

    def held(t, k):
        buf = torch.full((rows * (pitch + k) + 64,), 77.0, device="cuda", dtype=t.dtype)
        v = buf[shift + k:shift + k + rows * (pitch + k)].view(rows, pitch + k)[:, :d]
        v.copy_(t)
        return buf, v

    def untouched(buf, v, k):
        keep = buf.clone()
        keep[shift + k:shift + k + rows * (pitch + k)].view(rows, pitch + k)[:, :d] = 77
        return bool((keep == 77).all())

    for k in (0, 1):
        (_, xv), (yb, yv) = held(X, k), held(X, 0)
        rv, (sb, sv) = None if R is None else held(R, 2 * k)[1], held(X if R is None else R, k)
        got = ops.rms_norm(xv, G, EPS, residual=rv, out=yv, sum_out=None if R is None else sv, stats=True)
        assert got[0] is yv and (R is None or got[1] is sv)
        _check_forward(yv, None if R is None else sv, got[-1], X, R, G)
        assert untouched(yb, yv, 0) and (R is None or untouched(sb, sv, k))
        hs = X if R is None else sv
        dyv, dsv = held(dy, 1 - k)[1], None if ds is None else held(ds, 0)[1]
        _check_grad(*ops.rms_norm_backward(dyv, hs, got[-1], G, dsum=dsv), dy, hs, got[-1], G, ds)
        q = ops.rms_norm_fp8(xv, G, EPS, residual=rv)
        w = ops.rms_norm_fp8(X, G, EPS, residual=R)
        q, w = (q, w) if R is None else (q[0], w[0])
        differ = (q.codes.view(torch.uint8) != w.codes.view(torch.uint8)).float().mean()
        assert differ <= 0.002


@pytest.mark.parametrize("d", [130, 1031, 2048, 6000, 20001])
def test_in_place(d):
    torch, ops = _torch()
    X, R, G = _case(40, d, "bfloat16", "bfloat16", "float32", d)
    y, h, rstd = ops.rms_norm(X, G, residual=R, stats=True)
    for out, total in (("x", "r"), ("r", "x"), ("x", None), (None, "r"), (None, "x"), ("r", None)):
        x, r = X.clone(), R.clone()
        t = {"x": x, "r": r, None: None}
        got = ops.rms_norm(x, G, residual=r, out=t[out], sum_out=t[total], stats=True)
        assert torch.equal(got[0], y) and torch.equal(got[1], h) and torch.equal(got[2], rstd)
    x = X.clone()
    assert torch.equal(ops.rms_norm(x, G, out=x), ops.rms_norm(X, G))
    r = R.clone()
    q, hs = ops.rms_norm_fp8(X, G, residual=r, sum_out=r)
    w, _ = ops.rms_norm_fp8(X, G, residual=R)
    assert hs is r and torch.equal(r, h) and torch.equal(q.codes.view(torch.uint8), w.codes.view(torch.uint8))


@pytest.mark.parametrize("x,h", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", None)])
@pytest.mark.parametrize("d", [5, 8, 13, 35, 127, 128, 131, 250, 264, 500, 519, 1000, 1031, 2047, 4099, 6001, 8200, 16384, 16390])
def test_fp8_exactly_wherever_rows_start(d, x, h):
    """Two products, each rounded by itself, and the quantiser's codes: the same bits as torch's products with the rstd
    that was returned, then fp8_quantise.  Inputs and codes start anywhere, large values sit beside the groups' ends, and
    what lies between the rows of codes is not written."""
    torch, ops = _torch()
    from neuroflow_b200._nfx import lib
    rows, types = 9, {"float32": 0, "bfloat16": 1, "float16": 2}
    gen = torch.Generator(device="cuda").manual_seed(d)
    for shift, pitch, code_shift, code_pitch in ((0, d, 0, d), (1, d, 3, d + 1), (3, d + 1, 0, d + 7), (6, d + 2, 5, d), (7, d + 3, 1, d + 3),
                                                 (2, -(-d // 8) * 8, 4, -(-d // 16) * 16), (5, -(-d // 8) * 8 + 8, 6, d + 5)):
        def held(t):
            v = torch.zeros(rows * pitch + 16, device="cuda", dtype=t.dtype)[shift:shift + rows * pitch].view(rows, pitch)[:, :d]
            return v.copy_(t)
        X = torch.randn(rows, d, generator=gen, device="cuda")
        for i, c in enumerate((0, 6, 7, 120, 121, 127, 128, 129, 255, 256, d - 1)):
            if c < d:
                X[i % rows, c] = 1000.0 + i
        X[rows - 1, d // 2:] = 0
        X = held(X.to(getattr(torch, x)))
        R = None if h is None else held(torch.randn(rows, d, generator=gen, device="cuda").to(getattr(torch, h)))
        S = None if R is None else held(R)
        G = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
        groups = -(-d // 128)
        buf = torch.full((rows * code_pitch + 16,), 0x55, device="cuda", dtype=torch.uint8)
        scales, rstd = torch.empty(rows, groups, device="cuda"), torch.empty(rows, device="cuda")
        ptr = lambda t: None if t is None else t.data_ptr()
        assert lib.nfx_rms_norm_fp8(ptr(X), types[x], pitch, ptr(R), 0 if h is None else types[h], pitch, ptr(G), 0, rows, d, EPS,
                                    ptr(buf) + code_shift, code_pitch, ptr(scales), groups, 1, ptr(S), pitch, ptr(rstd),
                                    torch.cuda.current_stream().cuda_stream) == 0
        want, H, _ = _plain(X, R, G)
        assert S is None or torch.equal(S, H)
        q = ops.fp8_quantise((H.float() * rstd[:, None]) * G)
        codes = buf[code_shift:code_shift + rows * code_pitch].view(rows, code_pitch)[:, :d]
        assert torch.equal(codes, q.codes.view(torch.uint8)), (shift, pitch, code_shift, code_pitch)
        assert torch.equal(scales, q.scales)
        buf[code_shift:code_shift + rows * code_pitch].view(rows, code_pitch)[:, :d] = 0x55
        assert bool((buf == 0x55).all())


def test_empty_and_leading_dimensions():
    torch, ops = _torch()
    X, R, G = _case(12, 200, "float32", "float32", "float32", 1)
    y, h = ops.rms_norm(X.view(2, 3, 2, 200), G, residual=R.view(2, 3, 2, 200))
    assert y.shape == h.shape == (2, 3, 2, 200)
    assert torch.equal(y.view(12, 200), ops.rms_norm(X, G, residual=R)[0])
    one = torch.ones(200, device="cuda")
    assert torch.equal(ops.rms_norm(X, one), ops.rms_norm(X))
    e = X[:0]
    y, h, r = ops.rms_norm(e, G, residual=R[:0], stats=True)
    assert y.shape == (0, 200) and h.shape == (0, 200) and r.shape == (0,)
    dx, dres, dg = ops.rms_norm_backward(e, e, r, G)
    assert dx.shape == (0, 200) and torch.equal(dg, torch.zeros_like(G))
    q = ops.rms_norm_fp8(e, G)
    assert q.codes.shape == (0, 200)


@pytest.mark.parametrize("d", [64, 1031, 4096, 20001])
def test_bad_values_stay_in_their_row(d):
    """An infinity or a NaN makes its own row infinite or NaN by the formula, and no other."""
    torch, ops = _torch()
    X, R, G, dy, ds = _case(9, d, "bfloat16", "bfloat16", "float32", d, grad=True)
    y, h, rstd = ops.rms_norm(X, G, residual=R, stats=True)
    bad = X.clone()
    bad[2, d // 2], bad[5, d - 1] = float("nan"), float("inf")
    yb, hb, rb = ops.rms_norm(bad, G, residual=R, stats=True)
    keep = [i for i in range(9) if i not in (2, 5)]
    assert torch.equal(yb[keep], y[keep]) and torch.equal(rb[keep], rstd[keep])
    assert yb[2].isnan().all() and rb[5] == 0
    assert yb[5, d - 1].isnan() and (yb[5, :d - 1] == 0).all()  # inf * 0, and finite * 0
    g0, g1 = ops.rms_norm_backward(dy, h, rstd, G, dsum=ds), ops.rms_norm_backward(dy, hb, rb, G, dsum=ds)
    assert torch.equal(g1[0][keep], g0[0][keep]) and g1[0][2].isnan().all()
    q = ops.rms_norm_fp8(bad, G, residual=R)[0]
    w = ops.rms_norm_fp8(X, G, residual=R)[0]
    assert torch.equal(q.codes.view(torch.uint8)[keep], w.codes.view(torch.uint8)[keep])


def test_rows_of_zeros_and_eps():
    torch, ops = _torch()
    z = torch.zeros(3, 300, device="cuda")
    y, r = ops.rms_norm(z, eps=1e-4, stats=True)
    assert (y == 0).all() and ((r - 100).abs() < 1e-3).all()
    x = torch.full((3, 300), 1e-4, device="cuda")
    want = x.double() / (1e-8 + 1e-6) ** 0.5
    assert ((ops.rms_norm(x, eps=1e-6).double() / want - 1).abs() < 100 * EPS32).all()


def test_gradient_against_differences():
    """The directional derivative of sum(c y) + sum(e h), with y and h in fp32 as the forward kernels make
    them.  The difference quotient with step t is off by t^2 |third derivative| and by the rounding of the
    two sums over 2 t; 2e-3 of the gradient's size covers both here (t = 2^-6: t^2 / 6 = 4e-5 times curvatures of a
    few, and sums of 1,500 terms of size 1 to 2^-24 each over 2^-5: 1e-5)."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, res, g, c, e = rnd(5, 300), rnd(5, 300), 1 + 0.1 * rnd(300), rnd(5, 300), rnd(5, 300)
    ux, ur, ug = rnd(5, 300), rnd(5, 300), rnd(300)

    def f(t):
        y, h = ops.rms_norm(x + t * ux, g + t * ug, residual=res + t * ur)
        return float((c.double() * y.double()).sum() + (e.double() * h.double()).sum())

    t = 2.0 ** -6
    want = (f(t) - f(-t)) / (2 * t)
    for v in (x, res, g):
        v.requires_grad_()
    y, h = ops.rms_norm_autograd(x, g, residual=res)
    dx, dr, dg = torch.autograd.grad([y, h], [x, res, g], [c, e])
    got = float((dx.double() * ux).sum() + (dr.double() * ur).sum() + (dg.double() * ug).sum())
    size = float((dx.double() * ux).square().sum().sqrt() + (dr.double() * ur).square().sum().sqrt() + (dg.double() * ug).square().sum().sqrt())
    assert abs(got - want) <= 2e-3 * size


@pytest.mark.parametrize("x,h", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", None)])
def test_autograd(x, h):
    torch, ops = _torch()
    X, R, G, dy, ds = _case(31, 257, x, h, "float32", 5, grad=True)
    leaves = [t for t in (X, R, G) if t is not None]
    for t in leaves:
        t.requires_grad_()
    out = ops.rms_norm_autograd(X, G, EPS, residual=R)
    y, hs = (out, X.detach()) if R is None else (out[0], out[1].detach())
    want = ops.rms_norm(X.detach(), G.detach(), EPS, residual=None if R is None else R.detach(), stats=True)
    assert torch.equal(y.detach(), want[0])
    back = ops.rms_norm_backward(dy, hs, want[-1], G.detach(), dsum=ds)
    grads = torch.autograd.grad([y] if R is None else [y, out[1]], leaves, [dy] if R is None else [dy, ds])
    assert torch.equal(grads[0], back[0]) and torch.equal(grads[-1], back[2])
    if R is not None:
        assert torch.equal(grads[1], back[1]) and grads[1].dtype == R.dtype
        # only one of the outputs is used
        y, hh = ops.rms_norm_autograd(X, G, EPS, residual=R)
        a = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        b = ops.rms_norm_backward(dy, hs, want[-1], G.detach())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
        c = torch.autograd.grad(hh, leaves, ds, allow_unused=True)
        assert torch.equal(c[0], ds.to(X.dtype)) and torch.equal(c[1], ds) and (c[2] is None or not c[2].any())
        # gradients of two leaves do not share memory
        ops.rms_norm_autograd(X, G, EPS, residual=R)[0].float().sum().backward()
        assert X.grad.data_ptr() != R.grad.data_ptr()
    with torch.no_grad():
        again = ops.rms_norm_autograd(X, G, EPS, residual=R)
        assert not (again if R is None else again[0]).requires_grad
