"""The FP8 block quantiser, the FP8 block-scaled product and the linear layer made of them
(neuroflow_b200.ops / nfx_fp8_*) against plain implementations.

The quantiser is held bit for bit to a numpy restatement in which every fp32 rounding is written
out.  Products are compared with 64-bit ones of the same operands: with S = sum |a b| over K (scales
included), each block of 128 is summed by four tensor-core steps of 32 (fp32 results; 8 eps S_b
covers their alignment and rounding) and the ceil(K / 128) blocks are added in fp32 after two
roundings, so a result is off by at most (ceil(K / 128) + 12) eps S, eps = 2^-23, plus the
epilogue's few roundings and half an ulp of the output type.
"""
import numpy as np
import pytest

gpu = pytest.mark.gpu
EPS32 = 2.0 ** -23
ULP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _grid():
    """The non-negative E4M3 values in the order of their codes 0 .. 0x7E."""
    c = np.arange(0x7F)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))


def _encode(v):
    """E4M3 codes of float32 values: nearest, ties to the even code, under 2^-6 never above code 7."""
    grid = _grid()
    a = np.minimum(np.abs(v.astype(np.float64)), 448.0)
    nan = np.isnan(a)
    a = np.where(nan, 0.0, a)
    hi = np.clip(np.searchsorted(grid, a), 1, 0x7E)
    lo = hi - 1
    dl, dh = a - grid[lo], grid[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(a == grid[hi], hi, code)
    code = np.where((a < 2.0 ** -6) & (code > 7), 7, code)
    return np.where(nan, 0x7F, code | (np.signbit(v) << 7)).astype(np.uint8)


def _quantise(x, tile):
    """(codes, scales) of a float32 array, every rounding in float32."""
    r, k = x.shape
    h = 128 if tile else 1
    R, B = -(-r // h), -(-k // 128)
    p = np.zeros((R * h, B * 128), np.float32)
    p[:r, :k] = x
    c = p.reshape(R, h, B, 128)
    a = np.where(np.isfinite(c), np.abs(c), np.float32(0)).max((1, 3))
    s = np.maximum(a / np.float32(448), np.float32(2.0 ** -126)).astype(np.float32)
    inv = (np.float32(1) / s).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        codes = _encode((c * inv[:, None, :, None]).astype(np.float32)).reshape(R * h, B * 128)[:r, :k]
    return codes, s


def test_encoder_restatement():
    """The restatement gives every code back, and ties, carries and saturation where they belong."""
    g = _grid()
    assert np.array_equal(_encode(g.astype(np.float32)), np.arange(0x7F))
    assert np.array_equal(_encode(-g.astype(np.float32)), np.arange(0x7F) | 0x80)
    v = np.array([500, np.inf, -np.inf, np.nan, 1.0625, 1.1875, 7.6 / 512, 7.99 / 512, 447.9], np.float32)
    assert _encode(v).tolist() == [0x7E, 0x7E, 0xFE, 0x7F, 0x38, 0x3A, 7, 7, 0x7E]


def test_restatement_of_a_group():
    x = np.zeros((1, 130), np.float32)
    x[0, 3], x[0, 4], x[0, 129] = 896.0, -1.0, 0.5
    c, s = _quantise(x, False)
    assert s.tolist() == [[2.0, np.float32(0.5) / np.float32(448)]]
    assert c[0, 3] == 0x7E and c[0, 4] == 0xB0 and c[0, 129] == 0x7E and c[0, 0] == 0


def _case(r, c, dtype, seed):
    torch, _ = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(r, c, generator=g, device="cuda") * torch.exp(2 * torch.randn(1, c, generator=g, device="cuda"))
    return x.to(dtype)


def _bits(t):
    import torch
    return t.view(torch.uint8).cpu().numpy() if t.dtype != torch.uint8 else t.cpu().numpy()


def _same(q, x, tile):
    codes, s = _quantise(x, tile)
    assert np.array_equal(_bits(q.codes), codes)
    assert np.array_equal(q.scales.cpu().numpy().view(np.uint32), s.view(np.uint32))
    assert q.tile == tile and (q.codes.shape[0] < 2 or q.codes.stride(0) % 16 == 0)


SHAPES = [(1, 1), (33, 130), (7, 1002), (1, 128), (2, 127), (3, 129), (127, 16), (128, 128), (129, 257), (260, 384), (5, 4096), (513, 1000), (300, 7)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantise(shape, dtype):
    torch, ops = _torch()
    x = _case(*shape, getattr(torch, dtype), shape[0] * 31 + shape[1])
    xn = x.float().cpu().numpy()
    _same(ops.fp8_quantise(x), xn, False)
    _same(ops.fp8_quantise(x, tile=True), xn, True)
    for tile in (False, True):
        q, qt = ops.fp8_quantise(x, tile=tile, transposed=True)
        _same(q, xn, tile)
        _same(qt, np.ascontiguousarray(xn.T), tile)
    q, sums = ops.fp8_quantise(x, col_sums=True)
    q2, qt, sums2 = ops.fp8_quantise(x, transposed=True, col_sums=True)
    _same(q, xn, False), _same(q2, xn, False), _same(qt, np.ascontiguousarray(xn.T), False)
    want = xn.astype(np.float64).sum(0)
    assert np.all(np.abs(sums.cpu().numpy() - want) <= (shape[0] + 2) * 2.0 ** -24 * np.abs(xn).astype(np.float64).sum(0))
    assert torch.equal(sums, sums2)


@gpu
def test_quantise_special_values():
    """Zeros, the smallest and largest numbers, infinities and NaN: a bad element is encoded as
    such and the rest of its group keeps its scale."""
    torch, ops = _torch()
    x = np.random.default_rng(0).standard_normal((256, 300)).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 1e-45
    x[3] *= 1e-38
    x[4] *= 3e37
    x[5, 7], x[5, 200] = np.inf, -np.inf
    x[6, 9] = np.nan
    x[7] = np.nan
    x[8] = np.inf
    x[9, :128] = 2.0 ** -126
    t = torch.from_numpy(x).cuda()
    for tile in (False, True):
        q, qt = ops.fp8_quantise(t, tile=tile, transposed=True)
        _same(q, x, tile)
        _same(qt, np.ascontiguousarray(x.T), tile)
    _same(ops.fp8_quantise(t), x, False)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("pitch,shift", [(320, 0), (301, 0), (304, 1), (300, 8)])
def test_quantise_strides(dtype, pitch, shift):
    torch, ops = _torch()
    x = _case(200, 300, getattr(torch, dtype), 5)
    hold = torch.zeros(200 * pitch + 16, dtype=x.dtype, device="cuda")
    xs = hold[shift:shift + 200 * pitch].view(200, pitch)[:, :300]
    xs.copy_(x)
    xn = x.float().cpu().numpy()
    _same(ops.fp8_quantise(xs), xn, False)
    for tile in (False, True):
        q, qt = ops.fp8_quantise(xs, tile=tile, transposed=True)
        _same(q, xn, tile)
        _same(qt, np.ascontiguousarray(xn.T), tile)


@gpu
def test_quantise_long_offsets():
    torch, ops = _torch()
    x = _case(5, 200, torch.bfloat16, 6)
    pitch = 1 << 29
    wide = torch.empty(4 * pitch + 200, dtype=torch.bfloat16, device="cuda").as_strided((5, 200), (pitch, 1))
    wide.copy_(x)
    xn = x.float().cpu().numpy()
    _same(ops.fp8_quantise(wide), xn, False)
    q, qt = ops.fp8_quantise(wide, tile=True, transposed=True)
    _same(q, xn, True)
    _same(qt, np.ascontiguousarray(xn.T), True)


# ---- the product ----------------------------------------------------------------------------
def _operands(m, n, k, a_tile, b_tile, seed):
    torch, ops = _torch()
    a = ops.fp8_quantise(_case(m, k, torch.float32, seed), tile=a_tile)
    b = ops.fp8_quantise(_case(n, k, torch.float32, seed + 1) / max(k, 1) ** 0.5, tile=b_tile)
    return a, b


def _dense(q):
    s = q.scales.double().repeat_interleave(128, 1)[:, :q.codes.shape[1]]
    if q.tile:
        s = s.repeat_interleave(128, 0)[:q.codes.shape[0]]
    return q.codes.double() * s


def _gelu(z):
    import torch
    u = (2.0 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    return z * torch.sigmoid(2 * u)


def _check(got, a, b, bias=None, act=0):
    import torch
    A, B = _dense(a), _dense(b)
    k = A.shape[1]
    z, S = A @ B.t(), A.abs() @ B.abs().t()
    tol = (-(-k // 128) + 12) * EPS32 * S
    if bias is not None:
        z = z + bias.double()
        tol = tol + EPS32 * z.abs()
    if act == 1:
        # |gelu'| <= 1.13; the exponent's rounding enters as z gelu' terms, 16 eps |z| covers it
        tol = 1.2 * tol + 16 * EPS32 * z.abs()
        z = _gelu(z)
    elif act == 2:
        z = z.clamp_min(0)
    dt = str(got.dtype).replace("torch.", "")
    tiny = 2.0 ** -25 if dt == "float16" else 1e-37
    bad = (got.double() - z).abs() > tol + ULP[dt] * (z.abs() + tol) + tiny
    assert not bad.any(), (int(bad.sum()), tuple(got.shape), k)


MNK = [(1, 1, 1), (1, 128, 128), (1, 257, 1000), (2, 16, 4096), (7, 130, 129), (16, 512, 640), (17, 300, 127),
       (33, 1000, 2000), (64, 256, 384), (65, 129, 16), (127, 100, 257), (128, 128, 128), (129, 513, 900),
       (300, 70, 5000), (512, 512, 512), (1000, 3, 300), (777, 1111, 333), (2500, 2600, 200)]


@gpu
@pytest.mark.parametrize("mnk", MNK)
@pytest.mark.parametrize("tiles", [(False, True), (False, False), (True, True), (True, False)])
def test_gemm(mnk, tiles):
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    m, n, k = mnk
    a, b = _operands(m, n, k, *tiles, m + n + k)
    for dt in (torch.float32, torch.bfloat16):
        c = ops.fp8_gemm(a, b, out_dtype=dt)
        _check(c, a, b)
        assert torch.equal(c, ops.fp8_gemm(a, b, out_dtype=dt))
    assert _nfx.device_errors() == 0


@gpu
@pytest.mark.parametrize("m,n,k", [(3, 200, 500), (130, 300, 260), (900, 2000, 384), (4000, 1500, 128)])
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dt,bt", [("bfloat16", "bfloat16"), ("float32", "float32"), ("float16", "float32"), ("bfloat16", "float16")])
def test_gemm_epilogue(m, n, k, act, dt, bt):
    torch, ops = _torch()
    a, b = _operands(m, n, k, False, True, 3)
    bias = torch.randn(n, device="cuda").to(getattr(torch, bt))
    _check(ops.fp8_gemm(a, b, bias=bias, act=act, out_dtype=getattr(torch, dt)), a, b, bias, act)


@gpu
def test_gemm_integers_are_exact():
    """Unit scales and small integers: every sum is an integer below 2^24, so the result is exact and
    each element of K, block and tile is counted once."""
    torch, ops = _torch()
    g = torch.Generator(device="cuda").manual_seed(1)
    for m, n, k in [(1, 300, 1000), (40, 129, 515), (260, 520, 1100), (3000, 2100, 640)]:
        ints = [torch.randint(-8, 9, (r, k), generator=g, device="cuda").float() for r in (m, n)]
        ops_ = []
        for t, tile in zip(ints, (False, True)):
            r = t.shape[0]
            held = torch.zeros(r, -(-k // 16) * 16, device="cuda", dtype=torch.uint8)
            held[:, :k] = t.to(torch.float8_e4m3fn).view(torch.uint8)
            s = torch.ones(-(-r // 128) if tile else r, -(-k // 128), device="cuda")
            ops_.append(ops.Fp8Blocks(held.view(torch.float8_e4m3fn)[:, :k], s, tile))
        want = ints[0].double() @ ints[1].double().t()
        assert torch.equal(ops.fp8_gemm(*ops_, out_dtype=torch.float32).double(), want)
        swapped = ops.Fp8Blocks(ops_[1].codes, torch.ones(n, -(-k // 128), device="cuda"), False)
        assert torch.equal(ops.fp8_gemm(ops_[0], swapped, out_dtype=torch.float32).double(), want)


@gpu
def test_gemm_blocks_meet_their_scales():
    """Scales that are powers of two, another for each row, column tile and block, on codes of one:
    an exact result in which every scale can be told apart."""
    torch, ops = _torch()
    m, n, k = 200, 300, 700
    B = -(-k // 128)
    one = lambda r: torch.full((r, -(-k // 16) * 16), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :k]
    i = torch.arange
    sa = torch.ldexp(torch.ones(m, B), (i(m)[:, None] * 3 + i(B)) % 5).cuda()
    for rows, tile in ((-(-n // 128), True), (n, False)):
        sb = torch.ldexp(torch.ones(rows, B), (i(rows)[:, None] + 2 * i(B)) % 7).cuda()
        size = torch.tensor([min(128, k - 128 * b) for b in range(B)], device="cuda").double()
        full = sb.repeat_interleave(128, 0)[:n] if tile else sb
        want = (sa.double() * size) @ full.double().t()
        for scale in (sb, sb.t().contiguous().t()):
            c = ops.fp8_gemm(ops.Fp8Blocks(one(m), sa, False), ops.Fp8Blocks(one(n), scale, tile), out_dtype=torch.float32)
            assert torch.equal(c.double(), want)


@gpu
def test_gemm_bad_values_stay_in_their_row_and_column():
    torch, ops = _torch()
    for m in (5, 300):
        a, b = _operands(m, 260, 400, False, True, 9)
        clean = ops.fp8_gemm(a, b, out_dtype=torch.float32)
        a.codes.view(torch.uint8)[2, 399] = 0x7F
        b.codes.view(torch.uint8)[131, 0] = 0xFF
        c = ops.fp8_gemm(a, b, out_dtype=torch.float32)
        hit = torch.zeros_like(c, dtype=torch.bool)
        hit[2], hit[:, 131] = True, True
        assert c[hit].isnan().all() and torch.equal(c[~hit], clean[~hit])


@gpu
def test_gemm_output_strides_k_zero_and_empty():
    torch, ops = _torch()
    for m, n in ((9, 100), (257, 383)):
        a, b = _operands(m, n, 200, False, True, 4)
        bias = torch.randn(n, device="cuda")
        for dt in (torch.bfloat16, torch.float32):
            want = ops.fp8_gemm(a, b, bias=bias, out_dtype=dt)
            for pitch, shift in ((n + 1, 0), (n + 13, 1), (n + (-n) % 8 + 8, 0)):
                hold = torch.full((m * pitch + 8,), 55.0, dtype=dt, device="cuda")
                out = hold[shift:shift + m * pitch].view(m, pitch)[:, :n]
                assert ops.fp8_gemm(a, b, bias=bias, out=out) is out
                assert torch.equal(out, want)
                rest = hold[shift:shift + m * pitch].view(m, pitch)[:, n:]
                assert (rest == 55).all() and (hold[:shift] == 55).all() and (hold[shift + m * pitch:] == 55).all()
        none = ops.Fp8Blocks(a.codes[:, :0], a.scales[:, :0], False), ops.Fp8Blocks(b.codes[:, :0], b.scales[:, :0], True)
        c = ops.fp8_gemm(*none, bias=bias, act=2, out_dtype=torch.float32)
        assert torch.equal(c, bias.clamp_min(0).expand(m, n))
        assert ops.fp8_gemm(ops.Fp8Blocks(a.codes[:0], a.scales[:0], False), b).shape == (0, n)


@gpu
def test_gemm_rows_of_a_larger_matrix():
    """Operands that are slices: rows at a stride, an offset start, pad bytes that are not zero."""
    torch, ops = _torch()
    x, w = _case(300, 500, torch.float32, 1), _case(200, 500, torch.float32, 2)
    q, p = ops.fp8_quantise(x), ops.fp8_quantise(w)
    want = ops.fp8_gemm(q, p, out_dtype=torch.float32)
    hold = torch.full((600, 560), 0x55, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    codes = hold[::2, 32:532]
    codes.view(torch.uint8).copy_(q.codes.view(torch.uint8))
    assert torch.equal(ops.fp8_gemm(ops.Fp8Blocks(codes, q.scales, False), p, out_dtype=torch.float32), want)
    part = ops.Fp8Blocks(q.codes[40:50], q.scales[40:50], False)
    _check(ops.fp8_gemm(part, p, out_dtype=torch.float32), part, p)


@gpu
def test_gemm_long_offsets():
    """A result and an operand whose offsets pass 2^31 elements."""
    torch, ops = _torch()
    a, b = _operands(6, 300, 256, False, True, 8)
    want = ops.fp8_gemm(a, b, out_dtype=torch.bfloat16)
    pitch = 1 << 29
    out = torch.empty(5 * pitch + 300, dtype=torch.bfloat16, device="cuda").as_strided((6, 300), (pitch, 1))
    assert torch.equal(ops.fp8_gemm(a, b, out=out), want)
    codes = torch.empty(5 * pitch + 256, dtype=torch.uint8, device="cuda").as_strided((6, 256), (pitch, 1))
    codes.copy_(a.codes.view(torch.uint8))
    assert torch.equal(ops.fp8_gemm(ops.Fp8Blocks(codes, a.scales, False), b), want)


@gpu
def test_gemm_streams():
    torch, ops = _torch()
    a, b = _operands(700, 900, 1024, False, True, 12)
    want = ops.fp8_gemm(a, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [ops.fp8_gemm(a, b, stream=s) for s in streams for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(c, want) for c in got)


@gpu
def test_refusals():
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    a, b = _operands(8, 64, 256, False, True, 2)
    x = _case(8, 256, torch.float32, 1)
    bias = torch.zeros(64, device="cuda")
    B = ops.Fp8Blocks
    bad = [
        lambda: ops.fp8_quantise(x.cpu()),
        lambda: ops.fp8_quantise(x.double()),
        lambda: ops.fp8_quantise(x.t()),
        lambda: ops.fp8_quantise(x, tile=True, col_sums=True),
        lambda: ops.fp8_quantise(x[:1].expand(8, 256)),
        lambda: ops.fp8_gemm(a.codes, b),
        lambda: ops.fp8_gemm(B(a.codes[:, :128], a.scales[:, :1], False), b),
        lambda: ops.fp8_gemm(B(a.codes, a.scales[:, :1], False), b),
        lambda: ops.fp8_gemm(B(a.codes, a.scales.double(), False), b),
        lambda: ops.fp8_gemm(B(a.codes, a.scales, True), b),
        lambda: ops.fp8_gemm(B(a.codes.float(), a.scales, False), b),
        lambda: ops.fp8_gemm(a, b, bias=bias[:-1]),
        lambda: ops.fp8_gemm(a, b, act=3),
        lambda: ops.fp8_gemm(a, b, out_dtype=torch.float64),
        lambda: ops.fp8_gemm(a, b, out=torch.empty(8, 65, device="cuda")),
        lambda: ops.fp8_gemm(a, b, out=torch.empty(64, 8, device="cuda").t()),
        # rows that do not start on 16-byte boundaries: the copy engine's rule
        lambda: ops.fp8_gemm(B(torch.empty(8, 264, dtype=torch.uint8, device="cuda")[:, :256], a.scales, False), b),
        lambda: ops.fp8_gemm(B(torch.empty(8 * 256 + 16, dtype=torch.uint8, device="cuda")[8:8 + 2048].view(8, 256), a.scales, False), b),
        lambda: ops.fp8_linear(x, torch.zeros(64, 255, device="cuda")),
        lambda: ops.fp8_linear(x, torch.zeros(64, 256, device="cuda"), bias[:-1]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(_nfx.NfxError) as ei:
            f()
        assert ei.value.code == 1, i
    L = _nfx.lib
    c, s = a.codes.data_ptr(), a.scales.data_ptr()
    d, t = b.codes.data_ptr(), b.scales.data_ptr()
    o = torch.empty(8, 64, device="cuda").data_ptr()
    gemm = lambda m=8, n=8, k=256, p=c, act=0, ct=0, ldc=64: L.nfx_fp8_gemm(
        p, 256, s, 1, 8, 0, d, 256, t, 1, 1, 1, m, n, k, None, 0, act, o, ct, ldc, None)
    assert gemm(m=-1) == 1 and gemm(n=1 << 31) == 1 and gemm(act=-1) == 1 and gemm(ct=7) == 1 and gemm(ldc=7) == 1
    assert gemm(p=None) == 1 and gemm(p=c + 8) == 1
    assert gemm() == 0
    assert _nfx.device_errors() == 0


# ---- the linear layer -----------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("m,n,k,dtype", [(1, 64, 128, "bfloat16"), (37, 300, 200, "bfloat16"), (520, 256, 640, "float32"),
                                         (2, 3, 50, "float32"), (1000, 1030, 515, "bfloat16"), (130, 70, 260, "float16")])
def test_linear(m, n, k, dtype):
    """Output and gradients are the products of the dequantised operands; the same operands' product
    is linear in each, so its difference quotient along a direction is its derivative."""
    torch, ops = _torch()
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(m)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, b, dy = rnd(m, k).to(dt), (rnd(n, k) / k ** 0.5).to(dt), rnd(n).to(dt), rnd(m, n).to(dt)
    for t in (x, w, b):
        t.requires_grad_()
    y = ops.fp8_linear(x.view(1, m, k), w, b)
    assert y.shape == (1, m, n) and y.dtype == dt
    y.backward(dy.view(1, m, n))
    with torch.no_grad():
        xq, xt = ops.fp8_quantise(x, transposed=True)
        wq, wt = ops.fp8_quantise(w, tile=True, transposed=True)
        dq, dt_, sums = ops.fp8_quantise(dy, transposed=True, col_sums=True)
        assert torch.equal(_dense(wt), _dense(wq).t())
        _check(y.view(m, n), xq, wq, b)
        _check(x.grad, dq, wt)
        _check(w.grad, dt_, xt)
        assert torch.equal(b.grad, sums.to(dt))
        # f(X, W) = sum(dY . X W^T) with the gradient's own operands, along a direction in X and in W
        X, W, dY = _dense(xq), _dense(wq), _dense(dq)
        dX, h = rnd(m, k).double(), 0.5
        num = ((dY * ((X + h * dX) @ W.t())).sum() - (dY * ((X - h * dX) @ W.t())).sum()) / (2 * h)
        slack = lambda p, q, grad, d: (((-(-p.shape[1] // 128) + 12) * EPS32 * (p.abs() @ q.abs().t())
                                        + 2 * ULP[dtype] * grad.abs() + 2.0 ** -25) * d.abs()).sum() + 1e-9 * abs(num)
        assert abs(num - (x.grad.double() * dX).sum()) <= slack(dY, W.t(), x.grad.double(), dX)
        Xt, dYt = _dense(xt).t(), _dense(dt_).t()
        dW = rnd(n, k).double()
        num = ((dYt * (Xt @ (W + h * dW).t())).sum() - (dYt * (Xt @ (W - h * dW).t())).sum()) / (2 * h)
        assert abs(num - (w.grad.double() * dW).sum()) <= slack(dYt.t(), Xt.t(), w.grad.double(), dW)


@gpu
def test_linear_gradients_that_are_not_needed():
    torch, ops = _torch()
    x, w, b = _case(20, 96, torch.float32, 1), _case(40, 96, torch.float32, 2), torch.zeros(40, device="cuda")
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    ops.fp8_linear(*full).sum().backward()
    for need in range(1, 8):
        part = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b))]
        ops.fp8_linear(*part).sum().backward()
        for i, (p, f) in enumerate(zip(part, full)):
            assert (p.grad is None) if not need >> i & 1 else torch.equal(p.grad, f.grad)
    y = ops.fp8_linear(x, w)
    assert not y.requires_grad and torch.equal(y, ops.fp8_linear(x, w, b))


@gpu
def test_without_gradients():
    """Under no_grad the differentiable forms give the same outputs and record nothing."""
    torch, ops = _torch()
    x, w, b = _case(33, 200, torch.float32, 3), _case(70, 200, torch.float32, 4), torch.randn(70, device="cuda")
    g = torch.ones(200, device="cuda", requires_grad=True)
    for t in (x, w, b):
        t.requires_grad_()
    y, n = ops.fp8_linear(x, w, b), ops.layer_norm_autograd(x, g)
    assert y.requires_grad and n.requires_grad
    with torch.no_grad():
        y2, n2 = ops.fp8_linear(x, w, b), ops.layer_norm_autograd(x, g)
    assert not y2.requires_grad and not n2.requires_grad
    assert torch.equal(y, y2) and torch.equal(n, n2)
    assert torch.equal(n2, ops.layer_norm(x.detach(), g.detach()))


@gpu
def test_refusals_under_autograd():
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    x = _case(8, 64, torch.float32, 1).requires_grad_()
    for f in (lambda: ops.fp8_linear(x, torch.zeros(4, 63, device="cuda")), lambda: ops.fp8_linear(x.t(), torch.zeros(4, 8, device="cuda")),
              lambda: ops.layer_norm_autograd(x, torch.ones(63, device="cuda"))):
        with pytest.raises(_nfx.NfxError) as ei:
            f()
        assert ei.value.code == 1
