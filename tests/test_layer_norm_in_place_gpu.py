"""Layer norm with outputs in the place of inputs, as include/nfx.h allows: y in x, dx in x or in dy."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [96, 128, 771, 1030, 4096, 9998, 16384, 20001])
def test_outputs_in_place_of_inputs(d, dtype):
    import torch
    from neuroflow_b200 import _nfx, ops
    dt, rows = getattr(torch, dtype), 1301 if d < 8000 else 301
    gen = torch.Generator(device="cuda").manual_seed(d)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, dy, g = (rnd(rows, d) + 0.5).to(dt), rnd(rows, d).to(dt), 1 + 0.1 * rnd(d)
    y, mean, rstd = ops.layer_norm(x, g, stats=True)
    same = x.clone()
    assert ops.layer_norm(same, g, out=same) is same and torch.equal(same, y)
    dx, dg, db = ops.layer_norm_backward(dy, x, mean, rstd, g)
    n = _nfx.lib.nfx_layer_norm_backward_workspace(rows, d)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    kind = {"float32": 0, "bfloat16": 1}[dtype]
    for place in ("x", "dy"):
        t = {"x": x.clone(), "dy": dy.clone()}
        eg, eb = torch.empty_like(dg), torch.empty_like(db)
        rc = _nfx.lib.nfx_layer_norm_backward(t["dy"].data_ptr(), d, t["x"].data_ptr(), d, kind, mean.data_ptr(), rstd.data_ptr(),
                                              g.data_ptr(), 0, rows, d, t[place].data_ptr(), d, eg.data_ptr(), eb.data_ptr(),
                                              ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(t[place], dx) and torch.equal(eg, dg) and torch.equal(eb, db)
