"""Every tile form of the gated feed-forward block on whole numbers, where a missing, doubled or misplaced term of any sum changes the bits of a result."""
import pytest
import torch

from tests import gated_mlp_forms as gf

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
CASES = [(t, s) for t in TYPES for s in gf.FEW + gf.SIZES[t] + gf.KNOWN[t]]


@pytest.mark.parametrize("name,size", CASES, ids=[f"{t}-{'x'.join(map(str, s))}" for t, s in CASES])
def test_whole_numbers_are_exact(gpu_device, name, size):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    print(name, *size, flush=True)
    dtype = TYPES[name]
    *inp, dy = gf.whole_numbers(gpu_device, *size, dtype, seed=size[0])
    leaves = [t.requires_grad_(True) for t in inp]
    y = gated_mlp(*leaves, activation="relu")
    got = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    with torch.no_grad():
        got.append(gated_mlp(*leaves, activation="relu"))
        want = gf.exact(*leaves, dy, dtype)
    for n, a, b in zip(("y", "dx", "dw_gate", "dw_up", "dw_down", "y without gradients"), got, want + want[:1]):
        off = int((a != b).sum())
        assert off == 0, f"{n}: {off} of {b.numel()} entries differ"
        assert b.any()
