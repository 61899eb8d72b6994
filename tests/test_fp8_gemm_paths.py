"""The FP8 product on every path that its rule on sizes can choose: the kernel of CTA pairs, and the narrow
kernel with each tile width, with and without a split K and with each ring.  The CPU test holds the
shapes below to the rule, so that a change of the rule does not leave a path without a test; the GPU tests
compare each with the 64-bit product (tolerances as in test_fp8_block_gpu.py)."""
import ctypes as C

import pytest

from test_fp8_block_gpu import EPS32, ULP, _check, _dense, _operands, _torch

gpu = pytest.mark.gpu
B200_SMS = 148

# (columns, split, deep): (M, N, K); pairs last, with a K of several thousand, with a remainder
PATHS = {
    (16, 1, 1): (3, 91, 151), (16, 1, 0): (3, 19453, 151), (16, 2, 1): (269, 129, 1078), (16, 2, 0): (8, 19075, 4339),
    (16, 4, 1): (5, 91, 897), (16, 4, 0): (2, 19401, 13119), (16, 8, 1): (2, 91, 1942),
    (32, 1, 1): (826, 275, 154), (32, 1, 0): (19, 19023, 151), (32, 2, 1): (425, 259, 1684), (32, 2, 0): (18, 19111, 3750),
    (32, 4, 1): (260, 135, 932), (32, 4, 0): (18, 10389, 13269), (32, 8, 1): (131, 139, 2013),
    (64, 1, 1): (961, 515, 154), (64, 1, 0): (34, 19001, 164), (64, 2, 1): (629, 385, 2726), (64, 2, 0): (50, 19029, 3203),
    (64, 4, 1): (387, 273, 1882), (64, 4, 0): (35, 9473, 10625), (64, 8, 1): (267, 147, 3869),
    (128, 1, 1): (3221, 275, 152), (128, 2, 1): (788, 645, 2954), (128, 4, 1): (622, 401, 2436), (128, 8, 1): (362, 257, 5027),
    (0, 1, 0): (2301, 2043, 5007),
}
MORE = (0, 1, 4)  # further columns: rows that end elsewhere in 16 bytes
PAIRS = [(2501, 2603, 200), (2301, 2043, 5007), (1164, 1795, 152)]


def _plan(m, n, k, b_tile, sms=B200_SMS):
    from neuroflow_b200 import _nfx
    f = _nfx.lib.nfx_debug_fp8_gemm_plan
    f.restype = None
    f.argtypes = [C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int] + [C.POINTER(C.c_int)] * 3
    got = [C.c_int() for _ in range(3)]
    f(m, n, k, b_tile, sms, *got)
    return tuple(v.value for v in got)


def test_each_shape_takes_its_path():
    for path, (m, n, k) in PATHS.items():
        assert _plan(m, n, k, 1) == path and _plan(m, n, k, 0) == path, path
    for m, n, k in PAIRS:
        assert _plan(m, n, k, 0)[0] == 0 and all(_plan(m, n + more, k, 1)[0] == 0 for more in MORE)
    assert _plan(5, 40, 0, 1)[:2] == (16, 1)  # nothing to sum


def test_the_rule_on_devices_of_few_sms():
    """One SM (also what an unreadable count is taken for) has no pair, and none of them divides by zero."""
    assert _plan(2500, 2600, 200, 1, 0) == _plan(2500, 2600, 200, 1, 1) == _plan(2500, 2600, 200, 1, -5)
    for sms in (1, 2, 3, 7):
        for mnk in ((1, 1, 1), (1, 4096, 1 << 20), (2500, 2600, 200), (20000, 20000, 4096)):
            for b_tile in (0, 1):
                columns = _plan(*mnk, b_tile, sms)[0]
                assert columns in (16, 32, 64, 128) if sms == 1 else columns in (0, 16, 32, 64, 128)


def test_every_path_of_the_rule_has_a_shape():
    """A sweep over sizes meets no path that is not in the list, save narrow ones that differ in the split
    alone (a split of 8 in more CTAs than SMs)."""
    import random
    r = random.Random(0)
    known = {(c, min(s, 2), d) for c, s, d in PATHS}
    size = lambda top: int(round(top ** r.random()))
    for _ in range(20000):
        c, s, d = _plan(size(20000), size(30000), size(30000), r.randrange(2))
        assert (c, min(s, 2), d) in known


@gpu
@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("b_tile", [True, False])
def test_paths_against_64_bits(path, b_tile):
    torch, ops = _torch()
    from neuroflow_b200 import _nfx
    m, n, k = PATHS[path]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _plan(m, n, k, b_tile, sms) == path
    a, b = _operands(m, n, k, False, b_tile, m + k)
    bias = torch.randn(n, device="cuda")
    for dt, act, bb in ((torch.float32, 0, None), (torch.bfloat16, 2, bias)):
        c = ops.fp8_gemm(a, b, bias=bb, act=act, out_dtype=dt)
        _check(c, a, b, bb, act)
        assert torch.equal(c, ops.fp8_gemm(a, b, bias=bb, act=act, out_dtype=dt))
    assert _nfx.device_errors() == 0


@gpu
@pytest.mark.parametrize("mnk", PAIRS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_pairs_write_their_rows_and_nothing_else(mnk, dtype):
    """Row pitches and starts that allow copies of whole boxes, and ones that do not; rows that end inside
    16 bytes."""
    torch, ops = _torch()
    m, n, k = mnk
    dt = getattr(torch, dtype)
    for cols in (n + more for more in MORE):
        a, b = _operands(m, cols, k, False, True, 4)
        bias = torch.randn(cols, device="cuda")
        want = ops.fp8_gemm(a, b, bias=bias, out_dtype=dt)
        _check(want, a, b, bias)
        for pitch, shift in ((cols + 1, 0), (cols + 13, 1), (cols + (-cols) % 8 + 8, 0), (cols + (-cols) % 8, 8)):
            hold = torch.full((m * pitch + 16,), 55.0, dtype=dt, device="cuda")
            out = hold[shift:shift + m * pitch].view(m, pitch)[:, :cols]
            assert ops.fp8_gemm(a, b, bias=bias, out=out) is out
            assert torch.equal(out, want)
            rest = hold[shift:shift + m * pitch].view(m, pitch)[:, cols:]
            assert (rest == 55).all() and (hold[:shift] == 55).all() and (hold[shift + m * pitch:] == 55).all()


@gpu
@pytest.mark.parametrize("path", [p for p in PATHS if p[0] in (0, 64, 128)])
@pytest.mark.parametrize("b_tile", [True, False])
def test_bad_values_stay_in_their_row_and_column_on_each_path(path, b_tile):
    torch, ops = _torch()
    m, n, k = PATHS[path]
    a, b = _operands(m, n, k, False, b_tile, 9)
    clean = ops.fp8_gemm(a, b, out_dtype=torch.float32)
    row, col = m - 1, n - 2
    a.codes.view(torch.uint8)[row, k - 1] = 0x7F
    b.codes.view(torch.uint8)[col, 0] = 0xFF
    c = ops.fp8_gemm(a, b, out_dtype=torch.float32)
    hit = torch.zeros_like(c, dtype=torch.bool)
    hit[row], hit[:, col] = True, True
    assert c[hit].isnan().all() and torch.equal(c[~hit], clean[~hit])


@gpu
@pytest.mark.parametrize("path", [p for p in PATHS if p[0] in (0, 64, 128)])
def test_blocks_meet_their_scales_on_each_path(path):
    """Codes of one and scales that are powers of two, another for each row, column and block: every sum is a
    whole number below 2^24 and the result is exact."""
    torch, ops = _torch()
    m, n, k = PATHS[path]
    B = -(-k // 128)
    one = lambda r: torch.full((r, -(-k // 16) * 16), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :k]
    i = lambda r: torch.arange(r, device="cuda")
    pw = lambda e: torch.ldexp(torch.ones(e.shape, device="cuda"), e)
    sa = pw((i(m)[:, None] * 3 + i(B)) % 4)
    size = torch.tensor([min(128, k - 128 * b) for b in range(B)], device="cuda").double()
    for rows, tile in ((-(-n // 128), True), (n, False)):
        sb = pw((i(rows)[:, None] + 2 * i(B)) % 5)
        full = sb.repeat_interleave(128, 0)[:n] if tile else sb
        want = (sa.double() * size) @ full.double().t()
        assert want.max() < 2 ** 24
        c = ops.fp8_gemm(ops.Fp8Blocks(one(m), sa, False), ops.Fp8Blocks(one(n), sb, tile), out_dtype=torch.float32)
        assert torch.equal(c.double(), want)


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (130, 700, 900), (2501, 2603, 200)])
def test_capture_in_a_graph(m, n, k):
    """The operators of a layer, captured once and replayed on new contents of the same buffers."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(m)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, g, b, bias = rnd(m, k), 1 + 0.1 * rnd(k), 0.1 * rnd(k), rnd(n)
    w = ops.fp8_quantise(rnd(n, k) / k ** 0.5, tile=True)

    def layer():
        y, mean, rstd = ops.layer_norm(x, g, b, stats=True)
        z = ops.fp8_gemm(ops.layer_norm_fp8(x, g, b), w, bias=bias, act=1)
        q, qt, sums = ops.fp8_quantise(y, transposed=True, col_sums=True)
        return (y, z, q.codes.view(torch.uint8), q.scales, qt.codes.view(torch.uint8), qt.scales, sums,
                *ops.layer_norm_backward(y, x, mean, rstd, g))

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    for _ in range(2):
        x.copy_(rnd(m, k) + 0.3)
        graph.replay()
        want = layer()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
