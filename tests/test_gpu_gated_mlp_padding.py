"""The gated feed-forward block with dims that are no multiple of eight, beside infinities: what the dims are padded with adds nothing to the results."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _positive(dev, dtype, *shapes):
    gen = torch.Generator().manual_seed(5)
    return [(0.1 + torch.rand(*s, generator=gen)).to(dtype).to(dev) for s in shapes]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,D,F,Do", [(5, 61, 97, 39), (1, 1, 1, 1), (20, 8, 3, 8), (40, 1027, 41, 130), (70, 515, 127, 40), (300, 61, 97, 39), (600, 64, 513, 64)])
def test_an_infinite_row_is_infinite(gpu_device, M, D, F, Do, dtype, native):
    """Every operand positive: a row of x or dy with an infinity has an infinity in every result that it is in, and NaN in none."""
    from palimpsa_amd.ops.gated_mlp import _gated_mlp, gated_mlp
    call = gated_mlp if native else _gated_mlp
    x, wg, wu, wd, dy = _positive(gpu_device, dtype, (M, D), (F, D), (F, D), (Do, F), (M, Do))
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y0 = call(*leaves, "relu")
    (dx0,) = torch.autograd.grad(y0, leaves[:1], dy)
    row = M // 2
    rest = torch.arange(M, device=gpu_device) != row
    bad = x.detach().clone()
    bad[row, D // 2] = float("inf")
    y = call(bad, *leaves[1:], "relu")
    assert torch.isposinf(y[row]).all() and torch.equal(y[rest], y0[rest])
    with torch.no_grad():
        assert torch.equal(call(bad, *leaves[1:], "relu"), y)
    bad = dy.clone()
    bad[row, Do // 2] = float("inf")
    dx, dwg, dwu, dwd = torch.autograd.grad(call(*leaves, "relu"), leaves, bad)
    assert torch.isposinf(dx[row]).all() and torch.equal(dx[rest], dx0[rest])
    assert torch.isposinf(dwg).all() and torch.isposinf(dwu).all() and torch.isposinf(dwd[Do // 2]).all()
    others = torch.arange(Do, device=gpu_device) != Do // 2
    assert torch.isfinite(dwd[others]).all()
