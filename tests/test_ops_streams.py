"""What a call with `stream=` does with the tensors it is given, on the CPU with stand-ins for the
tensors, the stream and the compiled front-end, and on the GPU with the allocator's own behaviour."""
import contextlib

import pytest


class Held:
    """A tensor as `stream=` sees it: on the GPU, and told which streams use it."""
    is_cuda = True

    def __init__(self, device="cuda:0"):
        self.device, self.on = device, []

    def record_stream(self, s):
        self.on.append(s)


class Stream:
    def __init__(self, device="cuda:0"):
        self.device = device


@pytest.fixture
def ops(monkeypatch):
    from neuroflow_b200 import ops as m

    class Front:
        layer_norm = staticmethod(lambda *a: "y")
        layer_norm_fp8 = staticmethod(lambda *a: ("codes", "scales"))
        layer_norm_backward = staticmethod(lambda *a: ("dx", None, None))
        fp8_quantise = staticmethod(lambda *a: ("codes", "scales", None, None))
        fp8_gemm = staticmethod(lambda *a: "c")

    monkeypatch.setattr(m, "_ext", Front)
    monkeypatch.setattr(m.torch.cuda, "Stream", Stream)
    monkeypatch.setattr(m.torch.cuda, "stream", lambda s: contextlib.nullcontext())
    return m


def _calls(m, T):
    """Each operator, with every tensor that it reads or writes."""
    x, g, b, o, dy, mean, rstd, c, s, d, t = (T() for _ in range(11))
    return [
        (lambda st: m.layer_norm(x, g, b, out=o, stream=st), (x, g, b, o)),
        (lambda st: m.layer_norm(x, stream=st), (x,)),
        (lambda st: m.layer_norm_fp8(x, g, b, stream=st), (x, g, b)),
        (lambda st: m.layer_norm_backward(dy, x, mean, rstd, g, stream=st), (dy, x, mean, rstd, g)),
        (lambda st: m.fp8_quantise(x, stream=st), (x,)),
        (lambda st: m.fp8_gemm(m.Fp8Blocks(c, s), m.Fp8Blocks(d, t), bias=b, out=o, stream=st), (c, s, d, t, b, o)),
    ]


def test_tensors_of_a_call_are_recorded_on_its_stream(ops):
    """Their memory must not go to another tensor while the stream still uses it."""
    for call, used in _calls(ops, Held):
        for t in used:
            t.on.clear()
        st = Stream()
        call(st)
        assert all(t.on == [st] for t in used)


def test_streams_that_torch_does_not_own_are_not_recorded(ops, monkeypatch):
    """Memory recorded on a stream is looked after with an event on it when it is released; a stream of another
    library, wrapped or as a raw handle, may be gone by then."""
    class External(Stream):
        def __init__(self, handle, device=None):
            super().__init__(device)

    monkeypatch.setattr(ops.torch.cuda, "ExternalStream", External)
    for call, used in _calls(ops, Held):
        for st in (1234, External(1234, "cuda:0")):
            for t in used:
                t.on.clear()
            call(st)
            assert not any(t.on for t in used)


def test_a_stream_of_another_device_is_refused(ops):
    """It would be made current on its own device, and the call would run on another stream."""
    from neuroflow_b200 import _nfx
    for call, used in _calls(ops, Held):
        with pytest.raises(_nfx.NfxError) as ei:
            call(Stream("cuda:1"))
        assert ei.value.code == 1 and "cuda:1" in str(ei.value)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["layer_norm", "layer_norm_fp8", "layer_norm_backward", "fp8_quantise", "fp8_gemm"])
def test_inputs_released_while_the_stream_is_busy_keep_their_memory(which):
    import torch
    from neuroflow_b200 import ops
    x, w = torch.randn(64, 1000, device="cuda"), ops.fp8_quantise(torch.randn(96, 1000, device="cuda"), tile=True)
    g = torch.randn(1000, device="cuda")
    _, mean, rstd = ops.layer_norm(x, stats=True)

    def call(x, stream=None):
        if which == "layer_norm":
            return ops.layer_norm(x, g, stream=stream)
        if which == "layer_norm_fp8":
            return ops.layer_norm_fp8(x, g, stream=stream).dequantise()
        if which == "layer_norm_backward":
            return ops.layer_norm_backward(x, x, mean, rstd, g, stream=stream)[0]
        if which == "fp8_quantise":
            return ops.fp8_quantise(x, stream=stream).dequantise()
        return ops.fp8_gemm(x, w, stream=stream)

    make = (lambda: ops.fp8_quantise(x)) if which == "fp8_gemm" else x.clone
    tensors = lambda v: (v.codes, v.scales) if which == "fp8_gemm" else (v,)
    want = call(make())
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(make(), stream=s)  # (the stream's own memory is there: nothing below has to wait for an allocation)
    torch.cuda.synchronize()
    held = make()
    at = [t.untyped_storage().data_ptr() for t in tensors(held)]
    size = [t.untyped_storage().nbytes() for t in tensors(held)]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)  # some 50 ms, so that the call below is still to come
        got = call(held, stream=s)
    del held
    again = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for n in size]
    assert not {t.data_ptr() for t in again} & set(at)
    s.synchronize()
    assert torch.equal(got, want)
