"""The sums of a layer norm's dweight and dbias over the shares of its workgroups: in more bits than fp32 has."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,rows", [(64, 4096), (768, 2048), (4096, 512)])
def test_shares_that_cancel(gpu_device, D, rows):
    """A workgroup's rows sum to 2^27, another's to -2^27, and every other row adds one: fp32 would lose the ones beside the first.  Rows of plus and minus one in equal
    number are their own normalised rows, so dweight is as exact as dbias."""
    from palimpsa_amd.ops.layer_glue import layer_norm
    x = torch.ones(rows, D, device=gpu_device)
    x[:, 1::2] = -1
    dy = torch.ones_like(x)
    dy[:4], dy[-4:] = 0, 0
    dy[0], dy[-1] = 2.0 ** 27, -2.0 ** 27
    w, b = (torch.ones(D, device=gpu_device).requires_grad_(True) for _ in range(2))
    y = layer_norm(x, w, b, eps=0.0)
    assert torch.equal(y.detach(), x + 1)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    n = rows - 8
    assert (db == n).all()
    assert torch.equal(dw, n * x[0])
