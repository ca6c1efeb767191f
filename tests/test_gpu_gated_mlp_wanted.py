"""The gated feed-forward block with only some of its gradients wanted: the same numbers, and no kernel for what none of them needs."""
import pytest
import torch

from tests import feed_forward_bounds as fb
from tests.test_gpu_gated_mlp import make

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,D,F,Do", [(9, 64, 96, 72), (300, 61, 97, 39), (2000, 128, 512, 64)])
def test_only_the_last_weight_is_trained(gpu_device, M, D, F, Do, dtype, native):
    from palimpsa_amd import _lib as L
    from palimpsa_amd.ops.gated_mlp import _gated_mlp, gated_mlp
    *inp, dy = make(gpu_device, M, D, F, Do, dtype)
    call = (lambda *a: gated_mlp(*a)) if native else (lambda *a: _gated_mlp(*a, "silu"))
    wd = inp[3].clone().requires_grad_(True)
    y = call(*inp[:3], wd)
    torch.cuda.synchronize()
    L.profile_enable(True)
    try:
        (got,) = torch.autograd.grad(y, [wd], dy)
        torch.cuda.synchronize()
        seen = L.profile_read()
    finally:
        L.profile_enable(False)
    assert "mlp_dw" in seen and not {"mlp_grad", "mlp_dx"} & set(seen), seen
    val, tol = fb.gated_mlp(*inp, "silu", dtype, dy)
    fb.within(got, val["w_down"], tol["w_down"], "dw_down")
