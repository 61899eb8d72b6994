"""The operators of a pre-norm block in 16 bits used together: served, trained with clipping, on streams, under
autograd beyond a first backward pass, and what the calls refuse."""
import pytest

gpu = pytest.mark.gpu
pytestmark = gpu


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _params(d, hidden, seed, dtype):
    torch, _ = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    p = {"g1": 1 + 0.1 * rnd(d), "w1": (rnd(hidden, d) / d ** 0.5).to(dtype), "b1": 0.1 * rnd(hidden),
         "w2": (rnd(d, hidden) / hidden ** 0.5).to(dtype), "b2": 0.1 * rnd(d), "g2": 1 + 0.1 * rnd(d)}
    return p, rnd


def _block(ops, p, x, h):
    """h = x + h; h' = h + w2 gelu(w1 norm(h) + b1) + b2; the norm of h'."""
    n, h = ops.rms_norm_autograd(x, p["g1"], residual=h)
    y = ops.linear(ops.linear(n, p["w1"], p["b1"], act=1), p["w2"], p["b2"], residual=h)
    return ops.rms_norm_autograd(y, p["g2"])


def _plain(p, x, h):
    import torch
    norm = lambda v, g: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * g
    h = x + h
    a = torch.nn.functional.gelu(norm(h, p["g1"]) @ p["w1"].t() + p["b1"], approximate="tanh")
    return norm(a @ p["w2"].t() + p["b2"] + h, p["g2"])


@pytest.mark.parametrize("tokens,d,hidden", [(1, 64, 256), (77, 264, 1000), (600, 512, 2048)])
def test_block_and_its_gradients(tokens, d, hidden):
    """Against the block in 64 bits on the same 16-bit numbers.  Each of the six tensors on the way (sum, norm, hidden
    layer, output, and their gradients) is rounded to bf16, 2^-9 of its root mean square at random (2^-8 at most): a
    norm of the differences of at most 12 * 2^-8 of the result's (0.047), most of it unused."""
    torch, ops = _torch()
    p, rnd = _params(d, hidden, tokens, torch.bfloat16)
    x, h, c = rnd(tokens, d).bfloat16(), rnd(tokens, d).bfloat16(), rnd(tokens, d).bfloat16()
    leaves = [t.requires_grad_() for t in (*p.values(), x, h)]
    y = _block(ops, p, x, h)
    got = torch.autograd.grad(y, leaves, c)
    dp = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    dx, dh = x.detach().double().requires_grad_(), h.detach().double().requires_grad_()
    want_y = _plain(dp, dx, dh)
    want = torch.autograd.grad(want_y, [*dp.values(), dx, dh], c.double())
    assert float((y.double() - want_y).norm() / want_y.norm()) <= 12 * 2.0 ** -8
    for name, a, b, leaf in zip([*p, "x", "h"], got, want, leaves):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape
        assert float((a.double() - b).norm() / b.norm()) <= 12 * 2.0 ** -8, name


def test_training_step_clips_and_is_the_same_every_time():
    torch, ops = _torch()
    runs = []
    for _ in range(2):
        p, rnd = _params(128, 512, 3, torch.bfloat16)
        x, h, t = rnd(300, 128).bfloat16(), rnd(300, 128).bfloat16(), rnd(300, 128)
        for v in p.values():
            v.requires_grad_()
        opt = torch.optim.SGD(p.values(), lr=0.1)
        norms = []
        for _ in range(3):
            opt.zero_grad()
            ((_block(ops, p, x, h).float() - t) ** 2).mean().backward()
            before = torch.cat([v.grad.double().flatten() for v in p.values()]).norm()
            norms.append(ops.clip_grad_norm([v.grad for v in p.values()], 0.05))
            after = torch.cat([v.grad.double().flatten() for v in p.values()]).norm()
            assert abs(float(norms[-1]) / float(before) - 1) < 1e-5
            assert float(after) <= 0.05 * (1 + 2.0 ** -8)
            opt.step()
        runs.append([n.clone() for n in norms] + [v.detach().clone() for v in p.values()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_served_forms_agree_with_the_trained_ones():
    """Without gradients the same kernels run; with the norm in FP8 the linear layer is the FP8 one."""
    torch, ops = _torch()
    p, rnd = _params(256, 1024, 5, torch.bfloat16)
    for tokens in (1, 5, 300):
        x, h = rnd(tokens, 256).bfloat16(), rnd(tokens, 256).bfloat16()
        n, s = ops.rms_norm(x, p["g1"], residual=h)
        a = ops.gemm(n, p["w1"], bias=p["b1"], act=1)
        y = ops.rms_norm(ops.gemm(a, p["w2"], bias=p["b2"], residual=s), p["g2"])
        assert torch.equal(y, _block(ops, p, x, h))
        q, s8 = ops.rms_norm_fp8(x, p["g1"], residual=h)
        a8 = ops.fp8_gemm(q, ops.fp8_quantise(p["w1"], tile=True), bias=p["b1"], act=1)
        assert torch.equal(s8, s)
        # two operands rounded to FP8, 2^-4 of an element at most, at random: 2^-4 of the norm is far above
        assert float((a8.float() - a.float()).norm() / a.float().norm()) < 2.0 ** -4


@pytest.mark.parametrize("which", ["rms_norm", "rms_norm_fp8", "rms_norm_backward", "gemm", "gemm unaligned", "act_backward", "clip_grad_norm"])
def test_inputs_released_while_the_stream_is_busy_keep_their_memory(which):
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(64, 1000, generator=gen, device="cuda").bfloat16()
    w = torch.randn(96, 1000, generator=gen, device="cuda").bfloat16()
    odd = torch.randn(96, 1001, generator=gen, device="cuda").bfloat16()[:, :1000]
    g, rstd = torch.randn(1000, generator=gen, device="cuda"), torch.rand(64, generator=gen, device="cuda")
    fresh = torch.empty(64, 1000, device="cuda")

    def call(x, stream=None):
        if which == "rms_norm":
            return ops.rms_norm(x, g, residual=x, stream=stream)[0]
        if which == "rms_norm_fp8":
            return ops.rms_norm_fp8(x, g, stream=stream).dequantise()
        if which == "rms_norm_backward":
            return ops.rms_norm_backward(x, x, rstd, g, dsum=x, stream=stream)[0]
        if which == "act_backward":
            return ops.act_backward(x, x, 1, torch.float32, stream=stream)[1]
        if which == "clip_grad_norm":
            ops.clip_grad_norm([x], 1.0, out=[fresh], stream=stream)
            return fresh
        return ops.gemm(x, odd if "un" in which else w, stream=stream)

    want = call(x.clone()).clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(x.clone(), stream=s)  # (the stream's own memory is there: nothing below has to wait for an allocation)
    torch.cuda.synchronize()
    held = x.clone()
    at, size = held.untyped_storage().data_ptr(), held.untyped_storage().nbytes()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)  # some 50 ms, so that the call below is still to come
        got = call(held, stream=s)
    del held
    again = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    assert again.data_ptr() != at
    s.synchronize()
    assert torch.equal(got, want)


def _refused(f, word):
    from neuroflow_b200 import _nfx
    with pytest.raises(_nfx.NfxError) as ei:
        f()
    assert ei.value.code == 1 and word in str(ei.value), str(ei.value)


def test_second_derivatives_and_forward_mode_are_refused():
    torch, ops = _torch()
    import torch.autograd.forward_ad as fw
    p, rnd = _params(64, 96, 7, torch.bfloat16)
    x, h = rnd(20, 64).bfloat16(), rnd(20, 64).bfloat16()
    leaves = [t.requires_grad_() for t in (p["g1"], p["w1"], p["b1"], x, h)]
    forms = [(lambda: ops.rms_norm_autograd(x, p["g1"], residual=h)[0], (x, p["g1"], h)),
             (lambda: ops.rms_norm_autograd(x, p["g1"], residual=h)[1] * 1.0, (x, h)),
             (lambda: ops.linear(x, p["w1"], p["b1"], act=1, residual=None), (x, p["w1"], p["b1"]))]
    for f, params in forms:
        first = torch.autograd.grad((f().float() ** 2).sum(), params)
        for i in range(len(params)):
            y = f()
            grads = torch.autograd.grad((y.float() ** 2).sum(), params, create_graph=True)
            assert all(torch.equal(a.detach(), b) for a, b in zip(grads, first))
            _refused(lambda: (y.float().sum() + (grads[i].float() ** 2).sum()).backward(), "second")
        f().float().sum().backward(create_graph=True)
        for t in params:
            with torch.no_grad():
                t.grad.mul_(0.5)
            t.grad = None
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t.detach(), torch.ones_like(t))
        for f in (lambda: ops.rms_norm_autograd(dual(x), p["g1"]), lambda: ops.rms_norm_autograd(x, dual(p["g1"])),
                  lambda: ops.rms_norm_autograd(x, p["g1"], residual=dual(h)), lambda: ops.linear(dual(x), p["w1"]),
                  lambda: ops.linear(x, dual(p["w1"])), lambda: ops.linear(x, p["w1"], dual(p["b1"])),
                  lambda: ops.linear(x, p["w1"], None, residual=dual(rnd(20, 96).bfloat16()))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    _refused(f, "forward-mode")


def test_changed_saved_tensors_are_seen():
    """A tensor that the backward pass has saved is changed in place, by torch or by one of the calls."""
    torch, ops = _torch()
    p, rnd = _params(64, 96, 7, torch.bfloat16)
    x = rnd(20, 64).bfloat16().requires_grad_()
    buf = rnd(20, 64).bfloat16()
    w = p["w1"].clone().requires_grad_()
    y = ops.linear(buf, w, act=1)
    ops.rms_norm(x.detach(), out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    g = p["g1"].clone().requires_grad_()
    y, s = ops.rms_norm_autograd(x, g, residual=buf)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    leaf = torch.ones((), device="cuda", requires_grad=True)
    for write in (lambda t: ops.gemm(rnd(20, 64).bfloat16(), rnd(64, 64).bfloat16(), out=t),
                  lambda t: ops.rms_norm(rnd(20, 64).bfloat16(), residual=rnd(20, 64).bfloat16(), sum_out=t),
                  lambda t: ops.clip_grad_norm([t], 0.1), lambda t: ops.clip_grad_norm([rnd(20, 64)], 0.1, out=[t])):
        t = rnd(20, 64).bfloat16()
        loss = (t * leaf).sum()
        write(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            write(rnd(20, 64).bfloat16())


def test_refusals_of_the_front_end():
    torch, ops = _torch()
    rnd = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    x, r = rnd(20, 64), rnd(20, 64)
    pool = rnd(40 * 64)
    a, shifted = pool[:20 * 64].view(20, 64), pool[64:21 * 64].view(20, 64)
    _refused(lambda: ops.rms_norm(x, residual=r.half()), "residual")
    _refused(lambda: ops.rms_norm(x.float(), residual=r), "residual")
    _refused(lambda: ops.rms_norm(x, residual=r[:10]), "shape")
    _refused(lambda: ops.rms_norm(x, sum_out=r), "sum_out")
    _refused(lambda: ops.rms_norm(x, residual=r, sum_out=r.float()), "sum_out")
    _refused(lambda: ops.rms_norm(a, out=shifted), "shares memory")
    _refused(lambda: ops.rms_norm(x, residual=a, out=shifted), "shares memory")
    _refused(lambda: ops.rms_norm(x, residual=r, out=a, sum_out=shifted), "shares memory")
    _refused(lambda: ops.rms_norm(x, residual=r, out=x, sum_out=x), "shares memory")
    _refused(lambda: ops.rms_norm(x.t()), "contiguous")
    _refused(lambda: ops.rms_norm(x, torch.ones(63, device="cuda")), "gamma")
    _refused(lambda: ops.rms_norm(x, torch.ones(64)), "CUDA")
    _refused(lambda: ops.rms_norm(x[:, :0]), "empty")
    _refused(lambda: ops.rms_norm(x, eps=float("nan")), "eps")
    _refused(lambda: ops.rms_norm(x, out=torch.zeros_like(x, requires_grad=True)), "requires grad")
    _refused(lambda: ops.rms_norm_backward(x, r.half(), torch.ones(20, device="cuda")), "h must have")
    _refused(lambda: ops.rms_norm_backward(x, r, torch.ones(19, device="cuda")), "rstd")
    _refused(lambda: ops.rms_norm_backward(x, r, torch.ones(20, device="cuda"), dsum=r.float()), "dsum")
    w = rnd(32, 64)
    _refused(lambda: ops.gemm(x, w.half()), "b must be")
    _refused(lambda: ops.gemm(x.float(), w.float()), "a must be")
    _refused(lambda: ops.gemm(x, rnd(32, 63)), "columns")
    _refused(lambda: ops.gemm(x, w, bias=torch.ones(31, device="cuda")), "bias")
    _refused(lambda: ops.gemm(x, w, residual=rnd(20, 31)), "residual")
    _refused(lambda: ops.gemm(x, w, residual=torch.ones(20, 32, device="cuda")), "residual")
    _refused(lambda: ops.gemm(x, w, residual=rnd(32).expand(20, 32)), "overlap")
    _refused(lambda: ops.gemm(x, w, out_dtype=torch.float16), "Half")
    _refused(lambda: ops.gemm(x, w, act=3), "act")
    _refused(lambda: ops.gemm(x, w, act=1 << 32), "act")
    _refused(lambda: ops.gemm(x[:, ::2], w[:, ::2]), "contiguous")
    _refused(lambda: ops.gemm(x, w, out=torch.zeros(20, 32, device="cuda").bfloat16().requires_grad_()), "requires grad")
    sq = rnd(64, 64)
    _refused(lambda: ops.gemm(sq, w[:1].expand(64, 64) * 1, out=sq), "shares memory")
    _refused(lambda: ops.gemm(rnd(64, 64), sq, out=sq.t().contiguous().t()), "contiguous")
    _refused(lambda: ops.gemm(x, w, residual=pool[:640].view(20, 32), out=pool[32:672].view(20, 32)), "shares memory")
    wide = rnd(20, 128)  # side by side in wider rows: no element is shared
    assert torch.equal(ops.gemm(wide[:, :64], rnd(64, 64) * 0, out=wide[:, 64:]), torch.zeros(20, 64, device="cuda").bfloat16())
    _refused(lambda: ops.linear(x, w.half()), "weight")
    _refused(lambda: ops.linear(x, rnd(32, 63)), "weight")
    _refused(lambda: ops.linear(x, w, residual=rnd(20, 31)), "residual")
    _refused(lambda: ops.act_backward(x, None, 1), "z is needed")
    _refused(lambda: ops.act_backward(x, x.float(), 1), "z must")
    _refused(lambda: ops.clip_grad_norm([x, x], 1.0), "share memory")
    _refused(lambda: ops.clip_grad_norm([a, shifted], 1.0), "share memory")
    _refused(lambda: ops.clip_grad_norm([x, r], 1.0, out=[r, torch.empty_like(r)]), "shares memory")
    _refused(lambda: ops.clip_grad_norm([x], 1.0, out=[x, r]), "for each")
    _refused(lambda: ops.clip_grad_norm([x], 1.0, out=[r[:10]]), "shape")
    _refused(lambda: ops.clip_grad_norm([x], 1.0, out=[rnd(64, 20).t()]), "order")
    _refused(lambda: ops.clip_grad_norm([wide[:, :64]], 1.0), "contiguous")
    _refused(lambda: ops.clip_grad_norm([x], -1.0), "max_norm")
    _refused(lambda: ops.clip_grad_norm([x], float("nan")), "max_norm")
    _refused(lambda: ops.clip_grad_norm([x.requires_grad_()], 1.0), "require grad")
    _refused(lambda: ops.grad_norm([x.detach(), torch.zeros(3)]), "CUDA")
    assert ops.grad_norm(iter([r, r])).shape == ()  # (only read: the same tensor twice counts twice)


def test_backward_pass_in_a_graph():
    """Forward and backward captured together, after an eager pass over the same leaves whose graph is gone (one that
    lives ties the leaves to its stream, which torch refuses in a capture), and replayed."""
    torch, ops = _torch()
    p, rnd = _params(64, 96, 11, torch.bfloat16)
    x, h, c = rnd(30, 64).bfloat16(), rnd(30, 64).bfloat16(), rnd(30, 64).bfloat16()
    leaves = [t.requires_grad_() for t in (*p.values(), x, h)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(_block(ops, p, x, h), leaves, c)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(_block(ops, p, x, h), leaves, c)
    for _ in range(2):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        want = torch.autograd.grad(_block(ops, p, x, h), leaves, c)
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_rows_and_tensors_beyond_32_bit_offsets():
    """Rows 2^30 elements apart: the third one begins at element 2^31."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(12)
    pitch = 1 << 30
    hold = torch.zeros(2 * pitch + 4096, device="cuda", dtype=torch.bfloat16)

    def far(cols, at):
        v = hold.as_strided((3, cols), (pitch, 1), at)
        v.copy_(torch.randn(3, cols, generator=gen, device="cuda"))
        return v

    for cols in (300, 301):
        x, h, y, s = far(cols, 0), far(cols, 512), hold.as_strided((3, cols), (pitch, 1), 1024), hold.as_strided((3, cols), (pitch, 1), 1536)
        g = 1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")
        n, t, r = ops.rms_norm(x.contiguous(), g, residual=h.contiguous(), stats=True)
        a, b, q = ops.rms_norm(x, g, residual=h, out=y, sum_out=s, stats=True)
        assert torch.equal(a, n) and torch.equal(b, t) and torch.equal(q, r)
        u, v = ops.rms_norm_backward(x, s, q, g, dsum=h), ops.rms_norm_backward(x.contiguous(), t, q, g, dsum=h.contiguous())
        # dgamma: rows that lie otherwise go through another kernel, and each is within (rows + 4) 2^-24 sum |dy xh| of the
        # exact sum; dx's terms are rounded alike
        mag = (x.double() * s.double() * q.double()[:, None]).abs().sum(0)
        assert torch.equal(u[0], v[0]) and ((u[2].double() - v[2].double()).abs() <= 2 * 7 * 2.0 ** -24 * mag).all()
        c, e = ops.act_backward(x, h, 1, torch.float32), ops.act_backward(x.contiguous(), h.contiguous(), 1, torch.float32)
        assert torch.equal(c[0], e[0]) and torch.equal(c[1], e[1])
        # whole numbers, so that the sums are exact whichever kernel forms them
        for v in (x, h):
            v.copy_(torch.randint(-3, 4, (3, cols), generator=gen, device="cuda"))
        w = torch.randint(-3, 4, (200, cols), generator=gen, device="cuda").bfloat16()
        want = x.double() @ w.double().t()
        out = hold.as_strided((3, 200), (pitch, 1), 2048)
        assert torch.equal(ops.gemm(x, w, residual=h[:, :200], out=out), (want + h[:, :200].double()).bfloat16())
        assert torch.equal(ops.gemm(w, x, out_dtype=torch.float32).double(), want.t())
        assert torch.equal(ops.gemm(x.t(), x.t(), out_dtype=torch.float32).double(), x.double().t() @ x.double())


def test_operands_of_one_row_or_column_with_strides():
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(13)
    ints = lambda *s: torch.randint(-3, 4, s, generator=gen, device="cuda").bfloat16()
    for k in (1, 8, 70, 1000, 5000):
        for pitch in (1, 3, 8, 64):
            wide = ints(k, pitch)
            one = wide[:, :1].t()  # (1, k), k elements `pitch` apart
            other = ints(40, k)
            for a, b in ((one, other), (other, one), (one, one), (one, ints(k, 40).t()), (ints(k, 300).t(), one)):
                want = a.double() @ b.double().t()
                assert torch.equal(ops.gemm(a, b, out_dtype=torch.float32).double(), want), (k, pitch)
    a, b = ints(300, 1), ints(200, 1)
    assert torch.equal(ops.gemm(a, b, out_dtype=torch.float32).double(), a.double() @ b.double().t())


def test_linear_of_a_vector_and_of_no_tokens():
    torch, ops = _torch()
    p, rnd = _params(64, 96, 14, torch.bfloat16)
    w, b = p["w1"].requires_grad_(), p["b1"].requires_grad_()
    x = rnd(64).bfloat16().requires_grad_()
    for act in (0, 1, 2):
        y = ops.linear(x, w, b, act=act)
        assert y.shape == (96,) and torch.equal(y, ops.linear(x[None], w, b, act=act)[0])
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        ex, ew, eb = torch.autograd.grad(ops.linear(x[None], w, b, act=act), (x, w, b), torch.ones_like(y)[None])
        assert torch.equal(dx, ex) and torch.equal(dw, ew) and torch.equal(db, eb)
        none = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
        y = ops.linear(none, w, b, act=act, residual=torch.zeros(0, 96, device="cuda", dtype=torch.bfloat16))
        dx, dw, db = torch.autograd.grad(y, (none, w, b), torch.zeros_like(y))
        assert dx.shape == (0, 64) and not dw.any() and not db.any()
    y, h = ops.rms_norm_autograd(none, p["g1"].requires_grad_(), residual=none.detach())
    dg, = torch.autograd.grad(y, p["g1"], torch.zeros_like(y))
    assert y.shape == (0, 64) and not dg.any()


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("shape", [(3, 5, 64), (1, 64), (2, 1, 65), (4, 2, 3, 24)])
def test_linear_makes_the_gradients_that_are_asked_for(shape, act):
    """Any of the four gradients alone or together: the same bits, and those of the calls that the layer is made of."""
    torch, ops = _torch()
    gen = torch.Generator(device="cuda").manual_seed(act)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    k, n = shape[-1], 40
    ts = [rnd(*shape), rnd(n, k + 3)[:, :k], rnd(n), rnd(*shape[:-1], n)]
    dy = rnd(n, *shape[:-1]).movedim(0, -1)  # (not contiguous)
    x2, dy2 = ts[0].view(-1, k), dy.reshape(-1, n).contiguous()
    y, z = ops.gemm(x2, ts[1], bias=ts[2], act=act, residual=ts[3].reshape(-1, n), preact=True)
    dz, db = ops.act_backward(dy2, z, act, torch.bfloat16)
    want = [ops.gemm(dz, ts[1].t()).view(shape), ops.gemm(dz.t(), x2.t()), db, dy]
    for mask in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(ts)]
        got = ops.linear(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3])
        assert torch.equal(got.detach().view(-1, n), y)
        asked = [i for i in range(4) if mask >> i & 1]
        for i, g in zip(asked, torch.autograd.grad(got, [leaves[i] for i in asked], dy)):
            w = want[i]
            assert g.shape == ts[i].shape
            # (dz of one row may be taken as a row or a column: the same products, maybe added in another order)
            assert torch.equal(g, w) or (g.double() - w.double()).abs().max() <= 2.0 ** -8 * w.double().abs().max(), (mask, i)


def test_two_streams_at_once():
    """The same calls on two streams, without order between them: nothing is shared but the error word."""
    torch, ops = _torch()
    p, rnd = _params(256, 1000, 15, torch.bfloat16)
    xs = [rnd(700, 256).bfloat16() for _ in range(2)]
    odd = [rnd(33, 4001).bfloat16() for _ in range(2)]
    grads = [[rnd(n) for n in (5, 70001, 300)] for _ in range(2)]

    def work(i):
        n, h = ops.rms_norm(xs[i], p["g1"], residual=xs[1 - i])
        y = ops.gemm(ops.gemm(n, p["w1"], bias=p["b1"], act=1), p["w2"], residual=h)
        return [n, h, y, ops.gemm(odd[i], odd[1 - i]), ops.gemm(n.t(), y.t(), out_dtype=torch.float32),
                ops.rms_norm_backward(y, h, torch.ones(700, device="cuda"), p["g1"])[2], ops.grad_norm(grads[i])]

    want = [[t.clone() for t in work(i)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for _ in range(5):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i] = work(i)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
