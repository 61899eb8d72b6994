"""The 16-bit product on every path that its rule on sizes can choose: the kernels of CTA pairs without and with a
split K, the narrow kernel with each tile width, split and ring, and the kernel for few rows.  The CPU test holds
the shapes below to the rule, so that a change of the rule does not leave a path without a test; the GPU tests
compare each with whole numbers, whose sums are exact, and the epilogues with the 64-bit formula (tolerances as in
test_gemm_dense_gpu.py)."""
import ctypes as C

import pytest

from test_gemm_dense_gpu import _ints, _near, _torch, _want

gpu = pytest.mark.gpu
B200_SMS = 148

# (columns, split, deep): (M, N, K, A transposed); operands with rows on 16-byte boundaries, K and N that end elsewhere
PATHS = {
    (0, 1, 0): (1547, 657, 177, 1), (0, 2, 0): (830, 1417, 898, 1), (0, 4, 0): (897, 517, 2805, 1),
    (16, 1, 0): (1209, 131, 71, 0), (16, 1, 1): (20, 43, 84, 0), (16, 2, 0): (701, 337, 1107, 0), (16, 2, 1): (271, 137, 673, 0),
    (16, 4, 0): (295, 139, 454, 0), (16, 4, 1): (17, 43, 450, 0), (16, 8, 0): (161, 131, 1045, 0), (16, 8, 1): (18, 37, 993, 0),
    (32, 1, 0): (5191, 41, 70, 0), (32, 1, 1): (701, 389, 851, 0), (32, 2, 0): (345, 1565, 972, 0), (32, 2, 1): (680, 289, 1188, 0),
    (32, 4, 0): (386, 297, 1017, 0), (32, 4, 1): (268, 153, 1277, 0), (32, 8, 0): (104, 523, 993, 0), (32, 8, 1): (110, 131, 2449, 0),
    (64, 1, 0): (4982, 130, 93, 1), (64, 1, 1): (2, 38, 73, 1), (64, 2, 0): (831, 1367, 1231, 0), (64, 2, 1): (687, 290, 460, 1),
    (64, 4, 0): (802, 284, 474, 1), (64, 4, 1): (3, 38, 466, 1), (64, 8, 0): (302, 397, 1007, 1), (64, 8, 1): (3, 37, 1009, 1),
    (128, 1, 1): (1185, 956, 531, 1), (128, 2, 1): (925, 530, 863, 1), (128, 4, 1): (761, 278, 911, 1), (128, 8, 1): (274, 257, 1810, 1),
}
# further shapes: few rows or columns of a tile's second half, more tiles than pairs, a long K
MORE = [((16, 1, 0), (4355, 72, 130, 0)), ((64, 1, 0), (9000, 130, 40, 1)), ((0, 1, 0), (3100, 3000, 200, 0)), ((0, 2, 0), (512, 4096, 4097, 0)),
        ((0, 4, 0), (700, 700, 5000, 0)), ((128, 1, 1), (120, 16101, 1030, 0)), ((0, 1, 0), (12000, 72, 130, 0)), ((0, 1, 0), (19000, 130, 40, 1)),
        ((0, 1, 0), (120, 19101, 300, 0)), ((0, 1, 0), (12000, 72, 130, 1))]
# a long K in several runs, joined by a second kernel: (columns, split, deep, runs)
MORE += [((16, 8, 1, 2), (47, 214, 11781, 0)), ((16, 8, 1, 5), (17, 39, 10849, 0)), ((32, 8, 1, 3), (97, 10, 11997, 0)),
         ((64, 8, 1, 3), (194, 9, 8196, 1)), ((64, 8, 1, 13), (64, 64, 65536, 1)), ((128, 8, 1, 3), (202, 129, 11506, 0))]
# (split, B transposed, aligned): (M, N, K) of the kernel for few rows
FEW = {
    (1, 0, 0): [(2, 38, 70), (15, 37, 75), (32, 39, 76)], (1, 0, 1): [(2, 37, 70), (11, 38, 80), (1, 300, 9), (16, 41, 31)],
    (1, 1, 0): [(7, 43, 70), (11, 40, 73), (1, 64, 15)], (1, 1, 1): [(3, 42, 78), (10, 50, 75), (16, 200, 333), (1, 3, 16)],
    (2, 0, 0): [(6, 42, 2155), (9, 37, 845), (20, 46, 299)], (2, 0, 1): [(1, 38, 2556), (12, 39, 783)],
    (2, 1, 0): [(1, 44, 403), (11, 37, 407)], (2, 1, 1): [(1, 40, 411), (9, 45, 478)],
    (4, 0, 0): [(2, 41, 4184), (9, 37, 1549), (23, 45, 519)], (4, 0, 1): [(1, 39, 4166), (11, 40, 1680)],
    (4, 1, 0): [(1, 45, 784), (10, 42, 796)], (4, 1, 1): [(1, 41, 858), (11, 38, 1075)],
    (8, 0, 0): [(3, 49, 8456), (13, 43, 3370), (23, 39, 1058)], (8, 0, 1): [(5, 37, 8319), (12, 44, 3621)],
    (8, 1, 0): [(3, 37, 1652), (10, 38, 1708)], (8, 1, 1): [(2, 37, 1591), (10, 38, 1943)],
}


def _plan(m, n, k, a_t=0, b_t=0, aligned=1, sms=B200_SMS):
    from neuroflow_b200 import _nfx
    f = _nfx.lib.nfx_debug_gemm_plan
    f.restype = None
    f.argtypes = [C.c_int64] * 3 + [C.c_int] * 4 + [C.POINTER(C.c_int)] * 4
    got = [C.c_int() for _ in range(4)]
    f(m, n, k, a_t, b_t, aligned, sms, *got)
    return tuple(v.value for v in got[:3 if got[3].value == 1 else 4])  # (the runs of K where there are more)


def test_each_shape_takes_its_path():
    for path, (m, n, k, t) in PATHS.items():
        assert _plan(m, n, k, t) == path, path
    for path, (m, n, k, t) in MORE:
        assert _plan(m, n, k, t) == path, (path, m, n, k)
    for (split, b_t, aligned), shapes in FEW.items():
        for m, n, k in shapes:
            assert _plan(m, n, k, 0, b_t, aligned) == (-1, split, 0), (m, n, k)
    assert _plan(40, 40, 0)[1] == 1  # nothing to sum


def test_the_rule_on_devices_of_few_sms():
    """One SM (also what an unreadable count is taken for) has no pair, and none of them divides by zero."""
    assert _plan(2500, 2600, 200, sms=0) == _plan(2500, 2600, 200, sms=1) == _plan(2500, 2600, 200, sms=-5)
    for sms in (1, 2, 3, 7):
        for mnk in ((1, 1, 1), (40, 1, 1), (33, 4096, 1 << 20), (2500, 2600, 200), (20000, 20000, 4096)):
            for t in (0, 1):
                columns, split = _plan(*mnk, t, sms=sms)[:2]
                assert columns in ((-1, 16, 32, 64, 128) if sms == 1 else (-1, 0, 16, 32, 64, 128)) and split in (1, 2, 4, 8)


def test_every_path_of_the_rule_has_a_shape():
    import random
    r = random.Random(0)
    size = lambda top: int(round(top ** r.random()))
    for _ in range(20000):
        a_t = r.randrange(2)
        path = _plan(size(20000), size(30000), size(30000), a_t)
        assert path in PATHS or path[0] == -1 or (len(path) == 4 and path[1:3] == (8, 1) and path[0] in (16, 32, 64, 128)), path


def _held(rows, cols, fill, aligned=True, extra=0):
    """`fill` in rows that start on 16-byte boundaries, or not; what lies between them is NaN."""
    torch, _ = _torch()
    ld = -(-cols // 8) * 8 + extra + (0 if aligned else 3)
    buf = torch.full((rows * ld + 8,), float("nan"), device="cuda", dtype=fill.dtype)
    v = buf[0 if aligned else 1:][:rows * ld].view(rows, ld)[:, :cols]
    v.copy_(fill)
    return v


def _operands(m, n, k, a_t, b_t, dtype, seed, aligned=True):
    torch, _ = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    a, b = _ints(gen, m, k, dtype), _ints(gen, n, k, dtype)
    av = _held(k, m, a.t(), aligned).t() if a_t else _held(m, k, a, aligned)
    bv = _held(k, n, b.t(), aligned).t() if b_t else _held(n, k, b, aligned)
    return a, b, av, bv


@gpu
@pytest.mark.parametrize("path,shape", list(PATHS.items()) + MORE)
def test_paths_with_whole_numbers(path, shape):
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    m, n, k, a_t = shape
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _plan(m, n, k, a_t, sms=sms) == path
    for b_t in (0, 1):
        for dt in (torch.bfloat16, torch.float16):
            a, b, av, bv = _operands(m, n, k, a_t, b_t, dt, m + n)
            want = a.double() @ b.double().t()
            assert torch.equal(ops.gemm(av, bv, out_dtype=torch.float32).double(), want)
            bias, res = torch.arange(n, device="cuda").float() - 5, torch.ones(m, n, device="cuda").to(dt)
            got, z = ops.gemm(av, bv, bias=bias, act=2, residual=res, preact=True)
            assert torch.equal(z, (want + bias.double()).to(dt))
            assert torch.equal(got, ((want + bias.double()).clamp_min(0) + 1).to(dt))
    assert _nfx.device_errors() == 0


@gpu
@pytest.mark.parametrize("key", list(FEW))
def test_few_rows_with_whole_numbers(key):
    torch, ops = _torch()
    split, b_t, aligned = key
    for m, n, k in FEW[key]:
        for dt in (torch.bfloat16, torch.float16):
            a, b, av, bv = _operands(m, n, k, 0, b_t, dt, k, aligned)
            want = a.double() @ b.double().t()
            assert torch.equal(ops.gemm(av, bv, out_dtype=torch.float32).double(), want)
            bias, res = torch.arange(n, device="cuda").float() - 5, torch.ones(m, n, device="cuda").to(dt)
            got, z = ops.gemm(av, bv, bias=bias, act=2, residual=res, preact=True)
            assert torch.equal(z, (want + bias.double()).to(dt))
            assert torch.equal(got, ((want + bias.double()).clamp_min(0) + 1).to(dt))


@gpu
@pytest.mark.parametrize("path", [p for p in PATHS if p[0] in (0, 64) or p == (128, 1, 1)])
@pytest.mark.parametrize("out", ["bfloat16", "float32"])
def test_paths_against_64_bits(path, out):
    torch, ops = _torch()
    m, n, k, a_t = PATHS[path]
    gen = torch.Generator(device="cuda").manual_seed(k)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    a = _held(k, m, rnd(k, m).bfloat16()).t() if a_t else _held(m, k, rnd(m, k).bfloat16())
    b = _held(n, k, (2 * rnd(n, k) / k ** 0.5).bfloat16())
    ct = getattr(torch, out)
    bias, res = rnd(n).bfloat16(), rnd(m, n).to(ct)
    for act in (0, 1):
        want, tol, z, tz = _want(a, b, bias, act, res)
        got, zz = ops.gemm(a, b, bias=bias, act=act, residual=res, out_dtype=ct, preact=True)
        _near(got, want, tol)
        _near(zz, z, tz)
        assert torch.equal(got, ops.gemm(a, b, bias=bias, act=act, residual=res, out_dtype=ct))


@gpu
@pytest.mark.parametrize("shape", [PATHS[(0, 1, 0)], PATHS[(0, 2, 0)], PATHS[(0, 4, 0)], PATHS[(16, 2, 1)], PATHS[(128, 2, 1)], (12, 300, 500, 0),
                                   (47, 214, 11781, 0)])
@pytest.mark.parametrize("out", ["bfloat16", "float32"])
def test_results_of_any_pitch(shape, out):
    """Rows of C and of the residual that allow copies of whole boxes, and ones that do not; rows that end inside 16
    bytes; nothing beside the rows is written, and the residual may be C itself."""
    torch, ops = _torch()
    m, n, k, a_t = shape
    ct = getattr(torch, out)
    for cols in (n, n + 1, n + 4, (n + 7) // 8 * 8):
        a, b, av, bv = _operands(m, cols, k, a_t, 0, torch.bfloat16, 3)
        r = torch.arange(m, device="cuda")[:, None].remainder(13).to(ct).expand(m, cols).contiguous()
        want = (a.double() @ b.double().t() + r.double()).to(ct)
        for pitch, shift in ((cols + 1, 0), (cols + 13, 1), (cols + (-cols) % 8 + 8, 0), (cols + (-cols) % 8, 8)):
            hold = torch.full((m * pitch + 16,), 55.0, dtype=ct, device="cuda")
            c = hold[shift:shift + m * pitch].view(m, pitch)[:, :cols]
            assert ops.gemm(av, bv, residual=r, out=c) is c and torch.equal(c, want)
            c.copy_(r)
            assert ops.gemm(av, bv, residual=c, out=c) is c and torch.equal(c, want)
            rest = hold[shift:shift + m * pitch].view(m, pitch)[:, cols:]
            assert (rest == 55).all() and (hold[:shift] == 55).all() and (hold[shift + m * pitch:] == 55).all()


@gpu
@pytest.mark.parametrize("shape", [PATHS[(0, 1, 0)], PATHS[(0, 2, 0)], PATHS[(16, 2, 1)], PATHS[(64, 8, 1)], (12, 300, 500, 0), (5, 70, 33, 0),
                                   (47, 214, 11781, 0)])
def test_bad_values_stay_in_their_row_and_column(shape):
    torch, ops = _torch()
    m, n, k, a_t = shape
    for b_t in (0, 1):
        a, b, av, bv = _operands(m, n, k, a_t, b_t, torch.bfloat16, 9)
        clean = ops.gemm(av, bv, out_dtype=torch.float32)
        av[m - 1, k - 1], bv[n - 2, 0] = float("nan"), float("nan")
        got = ops.gemm(av, bv, out_dtype=torch.float32)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[m - 1], hit[:, n - 2] = True, True
        assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


@pytest.fixture
def budget():
    from neuroflow_b200 import _nfx
    f = _nfx.lib.nfx_debug_set_wait_budget_ns
    f.restype = None
    f.argtypes = [C.c_ulonglong]
    yield f
    f(0)


@gpu
@pytest.mark.parametrize("m,n,k", [(2048, 2304, 4096), (512, 4096, 4096), (64, 1024, 8192), (300, 700, 3000), (64, 64, 20000)])
def test_waits_that_run_out_are_reported(budget, m, n, k):
    """With a budget of 1 ns the pipeline waits give up, the kernel records it in the device error word, waits for its own
    copies and MMAs with the normal limit, releases its tensor memory and returns; with the normal budget the same
    context then computes the right result."""
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    gen = torch.Generator(device="cuda").manual_seed(k)
    a, b = torch.randn(m, k, generator=gen, device="cuda").bfloat16(), torch.randn(n, k, generator=gen, device="cuda").bfloat16()
    r = torch.randn(m, n, generator=gen, device="cuda").bfloat16()
    want = ops.gemm(a, b, residual=r)
    assert _nfx.device_errors() == 0
    budget(1)
    ops.gemm(a, b, residual=r)
    flags = _nfx.device_errors()  # synchronises; the launch itself succeeded
    assert flags != 0 and flags & ~0x1F == 0, hex(flags)
    budget(0)
    for _ in range(2):
        assert torch.equal(ops.gemm(a, b, residual=r), want)
        assert _nfx.device_errors() == 0


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (130, 700, 904), (333, 301, 77), (2501, 2604, 200)])
def test_capture_in_a_graph(m, n, k):
    """The operators of a block, captured once and replayed on new contents of the same buffers, between other calls on the
    same stream."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(m)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, h, g, bias = rnd(m, k).bfloat16(), rnd(m, k), 1 + 0.1 * rnd(k), rnd(n)
    w = (rnd(n, k) / k ** 0.5).bfloat16()

    def block():
        y, s, rstd = ops.rms_norm(x, g, residual=h, stats=True)
        c, z = ops.gemm(y, w, bias=bias, act=1, preact=True)
        dz, db = ops.act_backward(c, z, 1, torch.float32)
        dx, dw = ops.gemm(dz, w.t()), ops.gemm(dz.t(), y.t(), out_dtype=torch.float32)
        return (y, s, rstd, c, z, dz, db, dx, dw, *ops.rms_norm_backward(dx, s, rstd, g, dsum=s), ops.rms_norm_fp8(x, g, residual=h)[0].scales,
                ops.grad_norm([dw, db]))

    block()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block()
    for _ in range(2):
        x.copy_(rnd(m, k))
        h.copy_(rnd(m, k))
        graph.replay()
        want = block()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
