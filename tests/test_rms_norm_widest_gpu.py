"""The RMS norm and its gradient at the widest rows that they take, 2^31 - 257 columns, where a count of columns that is
stepped by a block's threads passes 2^31.  Tensors that start at unlike distances from a 16-byte boundary, as then
columns are taken one by one.

All elements are ones but for the last 2,000, which are twos: the mean of squares is 1 + 6000 / d = 1 + 2.8e-6.  A thread's
4.2 million terms and the joined sums are whole numbers; those beyond 2^24, the last few additions, are rounded by at
most 2^-24 each: 16 of them 1e-6.  The reciprocal root with eps = 0 is 1 within 2.5e-6, less than a bf16 step."""
import pytest

pytestmark = pytest.mark.gpu
D = (1 << 31) - 257
LAST = 2000


def _torch():
    import torch
    from neuroflow_b200 import ops
    return torch, ops


def _row(start, value=1.0):
    """A row of D elements `start` elements behind a 16-byte boundary."""
    torch, _ = _torch()
    x = torch.full((D + start,), value, device="cuda", dtype=torch.bfloat16)[start:]
    x[-LAST:] = 2 * value
    return x.view(1, D)


def _is(x, one, two, tol=0.0):
    for i in range(0, D - LAST, 1 << 28):
        assert ((x[0, i:min(i + (1 << 28), D - LAST)].float() - one).abs() <= tol).all(), i
    assert ((x[0, -LAST:].float() - two).abs() <= tol).all()


@pytest.fixture(autouse=True)
def room():
    torch, _ = _torch()
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_forward():
    torch, ops = _torch()
    before = (1 << 31) + 8
    hold = torch.full((before + D,), 7.0, device="cuda", dtype=torch.bfloat16)
    y, rstd = ops.rms_norm(_row(1), eps=0.0, out=hold[before:].view(1, D), stats=True)
    assert abs(float(rstd) - 1) <= 2.5e-6
    _is(y, 1, 2)
    assert (hold[:before] == 7).all()  # what lies in front of the row


def test_forward_into_fp8():
    """The largest value of a group is 448 as a code; a group of ones next to the twos has ones of 224 or 448."""
    torch, ops = _torch()
    got, h, rstd = ops.rms_norm_fp8(_row(0, 0.25), eps=0.0, residual=_row(1, 0.75), stats=True)
    assert abs(float(rstd) - 1) <= 2.5e-6
    _is(h, 1, 2)
    border = (D - LAST) // 128  # the group with both
    codes, scales = got.codes, got.scales
    want = torch.full((1, 1), 1 / 448, device="cuda")
    assert ((scales[:, :border] / want - 1).abs() <= 3e-6).all() and ((scales[:, border:] / (2 * want) - 1).abs() <= 3e-6).all()
    for i in range(0, border * 128, 1 << 28):
        assert (codes[0, i:min(i + (1 << 28), border * 128)].view(torch.uint8) == 0x7E).all(), i
    assert (codes[0, border * 128:D - LAST].view(torch.uint8) == 0x76).all() and (codes[0, D - LAST:].view(torch.uint8) == 0x7E).all()


def test_backward():
    """h all ones with rstd 1: dx = dy - mean(dy), dgamma = dy."""
    torch, ops = _torch()
    h = torch.ones(1, D, device="cuda", dtype=torch.bfloat16)
    dx, _, dgamma = ops.rms_norm_backward(_row(1), h, torch.ones(1, device="cuda"))
    _is(dx, 0, 1, 4e-6)
    _is(dgamma.view(1, D), 1, 2)
