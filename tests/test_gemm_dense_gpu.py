"""The 16-bit product with bias, activation and residual (neuroflow_b200.ops.gemm / nfx_gemm), the
activation's gradient and the linear layer against their formulas in 64 bits.

Tolerances.  Products of 16-bit numbers are exact in fp32.  Their sum is formed in fp32 in some order, by
units that may cut a sum off instead of rounding it, one step of 2^-23 of what is summed at most for each
addition: with s = sum |a b|, K 2^-23 s.  On top:
  bias, residual: a rounding each, 2^-24 of the result
  ReLU passes an error on; GELU multiplies one by at most 1.13 and has its own, |z| 2^-19: the exponent's
    argument 2u has a few roundings of 2^-24 of it, which moves the logistic function s by s (1 - s) |2u| 2^-22,
    at most 0.28 * 2^-22, and the hardware's exponential and division add a few 2^-22 of s
  the output type: half a step
Small whole numbers are summed without any rounding, so there the result is exact.
"""
import pytest

pytestmark = pytest.mark.gpu
EPS32 = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-38, "bfloat16": 1e-38, "float16": 2.0 ** -25}


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _gelu(z):
    import torch
    u = (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(2 * u)
    return z * s, s + z * s * (1 - s) * 2 * (2 / torch.pi) ** 0.5 * (1 + 0.134145 * z ** 2)


def _act(z, act):
    import torch
    if act == 1:
        return _gelu(z)
    if act == 2:
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).double()
    return z, torch.ones_like(z)


def _want(a, b, bias, act, res):
    """(result, its tolerance before the output's rounding, z, z's tolerance)"""
    k = a.shape[1]
    z = a.double() @ b.double().t()
    tz = k * 2.0 ** -23 * (a.double().abs() @ b.double().abs().t())
    if bias is not None:
        z = z + bias.double()
        tz = tz + EPS32 * z.abs()
    c, _ = _act(z, act)
    t = tz * (1.13 if act == 1 else 1.0) + (z.abs() * 2.0 ** -19 if act == 1 else 0)
    if res is not None:
        c = c + res.double()
        t = t + EPS32 * c.abs()
    return c, t, z, tz


def _near(got, want, tol):
    name = str(got.dtype)[6:]
    t = tol + HALF[name] * (want.abs() + tol) + TINY[name]
    bad = ~((got.double() - want).abs() <= t)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / t).max()))


def _ints(gen, rows, cols, dtype, top=3):
    import torch
    return torch.randint(-top, top + 1, (rows, cols), generator=gen, device="cuda").to(dtype)


SIZES = [(1, 1, 1), (1, 8, 8), (1, 4096, 512), (2, 3, 5), (3, 130, 64), (16, 64, 72), (17, 129, 40), (33, 257, 1000), (64, 128, 4104),
         (100, 1000, 136), (127, 255, 63), (128, 128, 64), (129, 513, 65), (200, 1024, 2048), (256, 256, 128), (257, 264, 200),
         (300, 700, 1543), (1000, 1000, 1000), (1025, 520, 72), (2100, 24, 72), (5, 2500, 3000), (2048, 2304, 320), (4097, 1032, 96)]


@pytest.mark.parametrize("layout", ["nn", "nt", "tn", "tt"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_whole_numbers_are_exact(m, n, k, layout):
    """Both operands in either order, sums below 2^24: every term is there, once."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    for dt in (torch.bfloat16, torch.float16):
        a = _ints(gen, m, k, dt) if layout[0] == "n" else _ints(gen, k, m, dt).t()
        b = _ints(gen, n, k, dt) if layout[1] == "n" else _ints(gen, k, n, dt).t()
        want = a.double() @ b.double().t()
        got = ops.gemm(a, b, out_dtype=torch.float32)
        assert got.dtype == torch.float32 and torch.equal(got.double(), want)
        assert torch.equal(ops.gemm(a, b), want.to(dt))


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dtype,out", [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("m,n,k", [(1, 1000, 512), (7, 33, 100), (64, 520, 1024), (130, 300, 264), (1100, 1000, 512), (2304, 2050, 192)])
def test_epilogue(m, n, k, dtype, out, act):
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(m + k + act)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    dt, ct = getattr(torch, dtype), getattr(torch, out)
    a, b = rnd(m, k).to(dt), (2 * rnd(n, k) / k ** 0.5).to(dt)
    for bias, res in ((rnd(n), None), (rnd(n).to(dt), rnd(m, n).to(ct)), (None, rnd(m, n).to(ct))):
        want, tol, z, tz = _want(a, b, bias, act, res)
        got = ops.gemm(a, b, bias=bias, act=act, residual=res, out_dtype=ct)
        _near(got, want, tol)
        c, zz = ops.gemm(a, b, bias=bias, act=act, residual=res, out_dtype=ct, preact=True)
        assert torch.equal(c, got) and zz.dtype == ct
        _near(zz, z, tz)
        assert torch.equal(got, ops.gemm(a, b, bias=bias, act=act, residual=res, out_dtype=ct))


@pytest.mark.parametrize("m,n,k", [(1, 300, 8192), (500, 300, 8192), (2304, 2304, 8192)])
def test_long_sums_in_fp32(m, n, k):
    """What a long sum of numbers of one sign loses: nothing like the bound above.  Random roundings of
    K / 16 steps give 2^-24 sqrt(K / 16) = 1.3e-6 of the sum, cut-off sums up to K / 16 2^-24 = 3e-5; sums
    joined from pieces of at most 512 terms stay below 32 * 2^-23 + 16 * 2^-24 = 4.8e-6."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(k)
    a = torch.rand(m, k, generator=gen, device="cuda").bfloat16()
    b = torch.rand(n, k, generator=gen, device="cuda").bfloat16()
    want = a.double() @ b.double().t()
    off = (ops.gemm(a, b, out_dtype=torch.float32).double() / want - 1).abs().max()
    assert off <= 4.8e-6, float(off)


@pytest.mark.parametrize("m,n,k", [(5, 40, 24), (130, 300, 200), (2304, 2050, 192), (300, 129, 1024)])
def test_strides_and_alignment(m, n, k):
    """Operands, residual and results whose rows start anywhere; what lies between the rows is not written."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(1)

    def held(rows, cols, pitch, shift, dt, fill=None):
        buf = torch.full((rows * pitch + shift,), 77.0, device="cuda", dtype=dt)
        v = buf[shift:].view(rows, pitch)[:, :cols]
        if fill is not None:
            v.copy_(fill)
        return buf, v

    for dt in (torch.bfloat16, torch.float16):
        a, b, r = _ints(gen, m, k, dt), _ints(gen, n, k, dt), _ints(gen, m, n, dt, 100)
        want = a.double() @ b.double().t() + r.double()
        for extra, shift in ((0, 0), (1, 0), (8, 8), (13, 3), (0, 1), (24, 16)):
            for t in (False, True):
                av = held(k, m, m + extra, shift, dt, a.t())[1].t() if t else held(m, k, k + extra, shift, dt, a)[1]
                bv = held(n, k, k + extra, shift, dt, b)[1] if t else held(k, n, n + extra, shift, dt, b.t())[1].t()
                rv = held(m, n, n + extra, shift, dt, r)[1]
                buf, cv = held(m, n, n + extra, shift, dt)
                assert ops.gemm(av, bv, residual=rv, out=cv) is cv
                assert torch.equal(cv, want.to(dt)), (extra, shift, t)
                keep = buf.clone()
                keep[shift:].view(m, n + extra)[:, :n] = 77
                assert (keep == 77).all()
                assert ops.gemm(av, bv, residual=rv, out=rv) is rv and torch.equal(rv, cv)  # added in place
                buf, cv = held(m, n, n + extra, shift, torch.float32)
                assert torch.equal(ops.gemm(av, bv, out=cv).double(), want - r.double())


def test_sizes_of_zero():
    torch, ops = _torch()
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)
    assert ops.gemm(z(0, 8), z(4, 8)).shape == (0, 4) and ops.gemm(z(3, 8), z(0, 8)).shape == (3, 0)
    bias = torch.randn(300, device="cuda")
    for m in (2, 300):
        r = torch.randn(m, 300, device="cuda").bfloat16()
        got, zz = ops.gemm(z(m, 0), z(300, 0), bias=bias, act=2, residual=r, preact=True)
        want = (bias.clamp_min(0) + r.float()).bfloat16()
        assert torch.equal(got, want) and torch.equal(zz, bias.bfloat16().expand(m, 300))


@pytest.mark.parametrize("m,n,k", [(3, 300, 200), (130, 300, 264), (2304, 2050, 192)])
def test_bad_values_stay_in_their_row_and_column(m, n, k):
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    a, b = rnd(m, k).bfloat16(), rnd(n, k).bfloat16()
    clean = ops.gemm(a, b, act=1)
    a[m - 1, k - 1], b[n - 2, 0] = float("nan"), float("inf")
    got = ops.gemm(a, b, act=1)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[m - 1], hit[:, n - 2] = True, True
    assert torch.equal(got[~hit], clean[~hit]) and got[m - 1].isnan().all()
    col = got[:m - 1, n - 2].float()
    want = torch.where(a[:m - 1, 0].float() > 0, float("inf"), 0.0)
    # gelu(inf) = inf, gelu(-inf) = 0 or NaN by the formula's -inf * 0
    assert torch.equal(col[want > 0], want[want > 0]) and (col[want == 0].isnan() | (col[want == 0] == 0)).all()


@pytest.mark.parametrize("z", [-3e38, -1e10, -100.0, -20.0, -7.0, -1.0, 0.0, 1e-30, 3.0, 50.0, 1e20, 3e38])
def test_gelu_far_out(z):
    """|z| 2^-19 covers the rounding where the function is not flat; far below zero the result is a zero."""
    torch, ops = _torch()
    a, b = torch.zeros(2, 8, device="cuda").bfloat16(), torch.zeros(40, 8, device="cuda").bfloat16()
    got = ops.gemm(a, b, bias=torch.full((40,), z, device="cuda"), act=1, out_dtype=torch.float32)
    want = float(_gelu(torch.tensor(z, device="cuda").double())[0]) if abs(z) < 1e5 else max(z, 0.0)
    tol = abs(z) * 2.0 ** -19 if z > -20 else 1e-20
    assert ((got.double() - want).abs() <= tol).all(), float(got[0, 0])


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 1000), (3, 257), (130, 64), (1000, 1031), (4100, 300)])
def test_act_backward(rows, cols, dtype, act):
    """dz: the slope has GELU's own error 2^-19 (its terms are of size one), a rounding, half a step; dbias: the
    rows' terms in any order, (rows + 2) 2^-24 of their sizes."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(rows)
    dt = getattr(torch, dtype)
    dy, z = (torch.randn(rows, cols, generator=gen, device="cuda").to(dt) for _ in range(2))
    z = (2 * z).to(dt)
    dz, db = ops.act_backward(dy, z, act, torch.float32)
    slope = _act(z.double(), act)[1]
    want = dy.double() * slope
    tol = dy.double().abs() * 2.0 ** -19 if act == 1 else want.abs() * 0
    _near(dz, want, tol)
    assert (dz is dy or torch.equal(dz, dy)) if act == 0 else dz.shape == dy.shape
    _near(db, want.sum(0), (tol + (rows + 2) * EPS32 * (want.abs() + tol)).sum(0))
    assert torch.equal(ops.act_backward(dy, z, act)[0], dz) and ops.act_backward(dy, z, act)[1] is None
    assert torch.equal(ops.act_backward(dy, z, act, torch.float32)[1], db)
    assert torch.equal(ops.act_backward(dy, z, act, torch.bfloat16)[1], db.bfloat16())


def test_act_backward_of_bad_and_far_values():
    torch, ops = _torch()
    z = torch.tensor([[-3e38, -1e5, -60.0, 0.0, 60.0, 1e5, 3e38, float("inf"), float("-inf"), float("nan")]], device="cuda")
    dy = torch.ones_like(z)
    g, _ = ops.act_backward(dy, z, 1)
    assert torch.equal(g[0, :3], torch.zeros(3, device="cuda")) and g[0, 3] == 0.5 and (g[0, 4:8] == 1).all()
    assert g[0, 8] == 0 and g[0, 9].isnan()
    r, _ = ops.act_backward(dy, z, 2)
    assert torch.equal(r[0, :9], torch.tensor([0, 0, 0, 0, 1, 1, 1, 1, 0.0], device="cuda")) and r[0, 9].isnan()


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("lead,k,n", [((1,), 64, 40), ((3, 5), 129, 257), ((300,), 512, 264), ((2304,), 264, 1000)])
def test_linear(lead, k, n, dtype, act):
    """Gradients of the layer: dz is off by its own rounding (half a step of the type), by z's (half a step of
    z, times the slope's own slope, at most 1.2) and by z's sum; both pass through the products."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    dt = getattr(torch, dtype)
    x, w, b = rnd(*lead, k).to(dt), (rnd(n, k) / k ** 0.5).to(dt), (0.2 * rnd(n))
    res, dy = rnd(*lead, n).to(dt), rnd(*lead, n).to(dt)
    leaves = (x, w, b, res)
    for t in leaves:
        t.requires_grad_()
    y = ops.linear(x, w, b, act=act, residual=res)
    dx, dw, db, dres = torch.autograd.grad(y, leaves, dy)
    X, W, B, D = x.detach().reshape(-1, k), w.detach(), b.detach(), dy.reshape(-1, n).double()
    want, tol, z, tz = _want(X, W, B, act, res.detach().reshape(-1, n))
    assert y.shape == (*lead, n) and y.dtype == dt
    _near(y.detach().reshape(-1, n), want, tol)
    slope = _act(z, act)[1]
    dz = D * slope
    near0 = (z.abs() <= tz) if act == 2 else torch.zeros_like(z, dtype=torch.bool)  # the sign may be either one
    h = HALF[dtype]
    tdz32 = D.abs() * ((2.0 ** -19 + 1.2 * (tz + h * z.abs() + TINY[dtype])) if act == 1 else 0) + D.abs() * near0
    tdz = tdz32 + ((dz.abs() + tdz32) * h + TINY[dtype] if act else 0)
    _near(dx.reshape(-1, k), dz @ W.double(), tdz @ W.double().abs() + n * 2.0 ** -23 * (dz.abs() @ W.double().abs()))
    r = X.shape[0]
    _near(dw, dz.t() @ X.double(), tdz.t() @ X.double().abs() + r * 2.0 ** -23 * (dz.abs().t() @ X.double().abs()))
    assert db.dtype == torch.float32
    _near(db, dz.sum(0), (tdz32 + (r + 2) * EPS32 * (dz.abs() + tdz32)).sum(0))
    assert torch.equal(dres, dy)
    with torch.no_grad():
        assert torch.equal(ops.linear(x, w, b, act=act, residual=res), y)


def test_linear_makes_only_the_gradients_that_are_asked_for():
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    x, w, b, r, dy = rnd(20, 64), rnd(24, 64), rnd(24), rnd(20, 24), rnd(20, 24)
    for act in (0, 1):
        full = None
        for needs in range(15, 0, -1):
            leaves = [t.detach().requires_grad_(bool(needs >> i & 1)) for i, t in enumerate((x, w, b, r))]
            asked = [t for t in leaves if t.requires_grad]
            got = dict(zip([i for i in range(4) if needs >> i & 1], torch.autograd.grad(ops.linear(*leaves[:3], act=act, residual=leaves[3]), asked, dy)))
            full = full or got
            assert all(torch.equal(g, full[i]) for i, g in got.items())


def test_linear_takes_strided_inputs():
    """Rows of a wider matrix, a transposed matrix, leading dimensions that are not evenly strided."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    w = rnd(40, 64)
    for x in (rnd(30, 100)[:, 20:84], rnd(64, 30).t(), rnd(5, 8, 64)[:, 1:7], rnd(6, 5, 64).transpose(0, 1)):
        a, b = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(), x.detach().requires_grad_()
        w1, w2 = w.clone().requires_grad_(), w.clone().requires_grad_()
        p, q = ops.linear(a, w1, act=1), ops.linear(b, w2, act=1)
        assert torch.equal(p, q)
        dy = rnd(*p.shape)
        for u, v in zip(torch.autograd.grad(p, (a, w1), dy), torch.autograd.grad(q, (b, w2), dy)):
            assert torch.equal(u, v)


def test_gradient_against_differences():
    """The directional derivative of sum(c y) in fp16 with the results' differences: a step t of the weights
    changes z by about t; the quotient is off by the outputs' rounding, 2^-12 of y's size in random directions over
    N = 40,000 results: 2^-12 sqrt(N) / (2 t), and by t^2 / 6 of the derivative.  With t = 1/4 (steps of the
    weights that fp16 holds exactly) that is 100 of a derivative of size sqrt(N K) ~ 1,600: 10 %."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(6)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    m, n, k = 200, 200, 64
    x, w, b, c = rnd(m, k).half(), (rnd(n, k) / 8).half(), rnd(n).half(), rnd(m, n).half()
    ub = c.float().sign().mean(0).sign()
    t = 0.25
    f = lambda s: float((c.double() * ops.linear(x, w, (b.float() + s * ub), act=1).double()).sum())
    want = (f(t) - f(-t)) / (2 * t)
    b.requires_grad_()
    db, = torch.autograd.grad(ops.linear(x, w, b, act=1), b, c)
    got = float((db.double() * ub.double()).sum())
    assert abs(got - want) <= 0.1 * max(abs(want), (m * n) ** 0.5)
