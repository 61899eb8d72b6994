"""The gradient norm and clipping (neuroflow_b200.ops.grad_norm, clip_grad_norm / nfx_grad_norm,
nfx_clip_grad_norm) against the formula in 64 bits.

Tolerances.  Squares are fp32 products at worst, added in fp32 over at most 64 elements of a thread and in 64
bits from there: 65 * 2^-24 of the sum of squares, half of that of the norm, and its rounding to fp32:
34 * 2^-24.  A scaled element has the scale's error, the scale's rounding, the product's and half a step of the
output type: 37 * 2^-24 and the half step."""
import pytest

pytestmark = pytest.mark.gpu
NORM = 34 * 2.0 ** -24
SCALE = 37 * 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -25}


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _norm(gs):
    import torch
    return float(sum((g.double().square().sum() for g in gs), torch.zeros((), dtype=torch.float64, device="cuda")).sqrt())


def _check(outs, before, norm, max_norm, eps=1e-6):
    want = _norm(before)
    assert norm.shape == () and str(norm.dtype) == "torch.float32"
    assert abs(float(norm) - want) <= NORM * want
    s = min(1.0, max_norm / (want + eps)) if want else 1.0
    for o, g in zip(outs, before):
        name = str(o.dtype)[6:]
        w = g.double() * s
        if s == 1.0:
            assert (o == g.to(o.dtype)).all()
        else:
            assert ((o.double() - w).abs() <= w.abs() * (SCALE + HALF[name] * (1 + 1e-3)) + TINY[name]).all()


def _grads(sizes, types, seed, size=1.0):
    torch, _ = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=gen, device="cuda") * size).to(getattr(torch, types[i % len(types)])) for i, n in enumerate(sizes)]


ALL = ("float32", "bfloat16", "float16")


@pytest.mark.parametrize("sizes", [[1], [2, 0, 3], [7, 4096, 1, 33], [100000], [16384, 16385, 16383], [5, 0, 0, 1000003], [0], [1] * 40])
@pytest.mark.parametrize("types", [("float32",), ("bfloat16",), ("float16",), ALL])
def test_in_place(sizes, types):
    torch, ops = _torch()
    g = _grads(sizes, types, len(sizes))
    before = [t.clone() for t in g]
    assert abs(float(ops.grad_norm(g)) - _norm(g)) <= NORM * _norm(g)
    assert all(torch.equal(p, q) for p, q in zip(g, before))
    for max_norm in (1e6, 0.7 * _norm(before), 0.0):
        g = [t.clone() for t in before]
        norm = ops.clip_grad_norm(g, max_norm)
        _check(g, before, norm, max_norm)
        assert torch.equal(norm, ops.grad_norm(before))


@pytest.mark.parametrize("src", ALL)
@pytest.mark.parametrize("dst", ALL)
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_into_other_tensors(src, dst, max_norm):
    """Views at every alignment of a flat buffer, of the other type."""
    torch, ops = _torch()
    sizes = [1, 3, 8, 5, 0, 4097, 64, 2, 16385, 9, 40000, 31, 7]
    g = _grads(sizes, (src,), 3)
    flat = torch.full((sum(sizes) + 3,), 5.0, device="cuda", dtype=getattr(torch, dst))
    out = list(flat[1:-2].split(sizes))
    before = [t.clone() for t in g]
    norm = ops.clip_grad_norm(g, max_norm, out=out)
    _check(out, before, norm, max_norm)
    assert all(torch.equal(p, q) for p, q in zip(g, before))
    assert flat[0] == 5 and (flat[-2:] == 5).all()
    # and from views of a flat buffer
    pool = torch.zeros(sum(sizes) + 3, device="cuda", dtype=getattr(torch, src))
    views = list(pool[3:].split(sizes))
    for v, t in zip(views, before):
        v.copy_(t)
    again = [torch.empty_like(o) for o in out]
    assert abs(float(ops.clip_grad_norm(views, max_norm, out=again)) / float(norm) - 1) <= 2 * NORM
    _check(again, before, norm, max_norm)


@pytest.mark.parametrize("count", [31, 33, 255, 257, 899, 900, 901, 2005])
def test_many_tensors(count):
    torch, ops = _torch()
    g = _grads([1 + 37 * i % 1000 for i in range(count)], ALL, count)
    before = [t.clone() for t in g]
    norm = ops.clip_grad_norm(g, 1.5)
    _check(g, before, norm, 1.5)
    assert torch.equal(ops.clip_grad_norm([t.clone() for t in before], 1.5), norm)


@pytest.mark.parametrize("size", [1e-37, 1e-30, 1e-15, 1e15, 1e19, 3e36])
def test_sizes_whose_squares_leave_fp32(size):
    torch, ops = _torch()
    g = _grads([1000, 3], ("float32",), 8, size)
    before = [t.clone() for t in g]
    norm = ops.clip_grad_norm(g, 0.5 * size, eps=0.0)
    _check(g, before, norm, 0.5 * size, 0.0)
    # beside ordinary ones, and beside zeros
    mixed = [torch.zeros(40000, device="cuda"), before[0], torch.ones(5, device="cuda")]
    assert abs(float(ops.grad_norm(mixed)) - _norm(mixed)) <= NORM * _norm(mixed)


def test_zeros_infinities_and_nan():
    torch, ops = _torch()
    z = [torch.zeros(100, device="cuda"), torch.zeros(0, device="cuda")]
    for max_norm, eps in ((1.0, 1e-6), (0.0, 0.0)):
        assert ops.clip_grad_norm(z, max_norm, eps) == 0 and not z[0].any()
    g = _grads([50, 60], ("float32",), 1)
    g[1][7] = float("inf")
    norm = ops.clip_grad_norm(g, 1.0)
    assert norm == float("inf") and not g[0].any() and g[1][7].isnan() and int(g[1].isnan().sum()) == 1
    g = _grads([50, 60], ("bfloat16",), 1)
    g[1][7] = float("nan")
    assert ops.grad_norm(g).isnan()
    assert ops.clip_grad_norm(g, 1.0).isnan() and all(t.isnan().all() for t in g)
    # a largest norm of infinity leaves everything as it is
    g = _grads([50], ("float32",), 2)
    w = g[0].clone()
    ops.clip_grad_norm(g, float("inf"))
    assert torch.equal(g[0], w)


def test_a_sum_beyond_fp32_is_scaled_all_the_same():
    """The norm is infinite as an fp32 number, the scale is not taken from that number."""
    torch, ops = _torch()
    g = [torch.full((100,), 3e38, device="cuda")]
    norm = ops.clip_grad_norm(g, 1.0)
    assert norm == float("inf")
    assert ((g[0].double() - 0.1).abs() <= 0.1 * SCALE).all()


@pytest.mark.parametrize("count", [47, 48, 49, 239, 240, 241, 899, 900, 901, 1805])
def test_lists_as_long_as_the_tables(count):
    """Lists that just fit a table of the kernels' parameters or just do not, some tensors without elements among them,
    in place and into unaligned parts of one buffer."""
    torch, ops = _torch()
    g = _grads([(37 * i) % 900 * (i % 7 != 3) + 2000 * (i % 50 == 0) for i in range(count)], ALL, count)
    before = [t.clone() for t in g]
    assert abs(float(ops.grad_norm(g)) - _norm(g)) <= NORM * _norm(g)
    flat = torch.full((sum(t.numel() for t in g) + 3,), 7.0, device="cuda")
    out = list(flat[1:-2].split([t.numel() for t in g]))
    _check(out, before, ops.clip_grad_norm(g, 2.0, out=out), 2.0)
    assert all(torch.equal(p, q) for p, q in zip(g, before)) and flat[0] == 7 and (flat[-2:] == 7).all()
    _check(g, before, ops.clip_grad_norm(g, 2.0), 2.0)


def test_permuted_and_large():
    torch, ops = _torch()
    a = _grads([64 * 48], ("float32",), 4)[0].view(64, 48)
    g = [a.clone().t(), a.clone().view(4, 16, 48).permute(2, 0, 1)]
    before = [t.clone() for t in g]
    _check(g, before, ops.clip_grad_norm(g, 2.0), 2.0)
    out = [torch.empty(48, 64, device="cuda", dtype=torch.bfloat16).t().contiguous().t()]
    out = [torch.empty(64, 48, device="cuda", dtype=torch.bfloat16).t()]
    ops.clip_grad_norm([before[0]], 2.0, out=out)
    _check(out, before[:1], ops.grad_norm(before[:1]), 2.0)
    big = _grads([(1 << 25) + 5, 3, 1 << 22], ("bfloat16", "float32"), 5, 0.01)
    before = [t.clone() for t in big]
    _check(big, before, ops.clip_grad_norm(big, 1.0), 1.0)


def test_elements_beyond_32_bits():
    """A tensor of 2^31 and more elements: ones, some of them twos near the end."""
    torch, ops = _torch()
    n = (1 << 31) + 1000
    g = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    g[-500:] = 2
    want = float(n + 500 * 3) ** 0.5
    norm = ops.clip_grad_norm([g], want / 2, eps=0.0)
    assert abs(float(norm) - want) <= NORM * want
    assert (g[:1000] == 0.5).all() and (g[n - 1000:n - 500] == 0.5).all() and (g[-500:] == 1).all()
    assert int((g == 0.5).sum()) == n - 500


def test_capture_in_graphs_that_share_memory():
    """Two captured calls replayed in turn on new gradients: neither disturbs the other."""
    torch, ops = _torch()
    a, b = _grads([1000, 70000], ALL, 1), _grads([33, 5, 20000], ALL, 2)
    oa, ob = [torch.empty(t.shape, device="cuda") for t in a], [torch.empty(t.shape, device="cuda") for t in b]
    ops.clip_grad_norm(a, 1.0, out=oa)
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga, pool=pool):
        na = ops.clip_grad_norm(a, 1.0, out=oa)
    with torch.cuda.graph(gb, pool=pool):
        nb = ops.clip_grad_norm(b, 2.0, out=ob)
    for seed in (11, 12):
        for t, s in zip(a + b, _grads([1000, 70000], ALL, seed) + _grads([33, 5, 20000], ALL, seed + 5)):
            t.copy_(s)
        ga.replay()
        gb.replay()
        ga.replay()
        _check(oa, a, na.clone(), 1.0)
        gb.replay()
        _check(ob, b, nb.clone(), 2.0)


@pytest.mark.parametrize("count", [2, 60, 250, 901])
@pytest.mark.parametrize("n", [50, 40000])
def test_a_largest_norm_of_infinity_with_an_infinite_element(count, n):
    """Nothing is scaled, in place or into other tensors; a NaN makes NaN of everything all the same."""
    torch, ops = _torch()
    inf = float("inf")
    g = _grads([n] + [5] * (count - 1), ALL, 1)
    g[0][7], g[1][2] = inf, -inf
    before = [t.clone() for t in g]
    out = [torch.zeros(t.shape, device="cuda") for t in g]
    assert ops.clip_grad_norm(g, inf, out=out) == inf and all(torch.equal(o, t.float()) for o, t in zip(out, before))
    assert ops.clip_grad_norm(g, inf) == inf and all(torch.equal(t, b) for t, b in zip(g, before))
    g[1][3] = float("nan")
    assert ops.clip_grad_norm(g, inf).isnan() and all(t.isnan().all() for t in g)


@pytest.mark.parametrize("dtype,group", [("float32", 16), ("bfloat16", 32), ("float16", 32)])
@pytest.mark.parametrize("sizes", [[33], [5000] * 7, [1 << 20, 3]])
def test_norm_within_what_a_group_of_squares_loses(sizes, dtype, group):
    """A group's additions are off by 2^-24 of its sum each at most; the groups, positive all of them, are added in 64 bits, so
    the sum of squares is off by group 2^-24 of itself, the norm by half of that and its rounding to fp32."""
    torch, ops = _torch()
    for size in (1.0, 1e-3, 300.0):
        g = _grads(sizes, (dtype,), group, size)
        want = _norm(g)
        assert abs(float(ops.grad_norm(g)) - want) <= (group / 2 + 1) * 2.0 ** -24 * want
