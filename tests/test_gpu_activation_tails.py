"""Activations of the gated feed-forward block far below zero, where they are small: right in proportion to themselves, not to the other entries."""
import pytest
import torch

from oracle import feed_forward_oracle as fo
from tests import feed_forward_bounds as fb

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24


def _exact(act, g):
    if act != "gelu_tanh":
        return fo.activation(act, g)
    # (1 + tanh(z / 2)) / 2 as the logistic function of z: beyond z = -30 the sum is 2^-43 and less, and 64 bits of it hold no ten
    z, dz = (8 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3), (8 / torch.pi) ** 0.5 * (1 + 0.134145 * g * g)
    f = torch.sigmoid(z)
    return g * f, f + g * f * (1 - f) * dz


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M", [12, 40, 1000])
def test_small_values_keep_their_bits(gpu_device, act, M):
    """Seven hidden entries that are entries of x, the eighth entry of x being one: y are the activations and dx their derivatives, each a single product."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    t = -torch.linspace(0.5, 12.5 if act != "gelu_tanh" else 7.0, 7 * M, device=gpu_device).reshape(M, 7)     # (gelu_tanh falls as e^(-0.07 |g|^3))
    x = torch.cat([t, torch.ones(M, 1, device=gpu_device)], 1).requires_grad_(True)
    eye = torch.eye(8, device=gpu_device)
    wg, wu, wd = torch.diag(torch.tensor([1.] * 7 + [0.], device=gpu_device)), torch.zeros(8, 8, device=gpu_device), eye
    wu[:7, 7] = 1
    y = gated_mlp(x, wg, wu, wd, act)
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    a, d = _exact(act, t.double())
    # The argument z of the exponential is off by a few roundings of itself, and the exponential by that: |z| is g, g^2 / 2 or 1.6 |g| (1 + 0.045 g^2).  What
    # stands before it (erfc's fraction by 16 units, reciprocals, products) by 40 roundings.
    z = {"silu": t.abs(), "gelu": t * t / 2, "gelu_tanh": 1.6 * t.abs() * (1 + 0.045 * t * t)}[act].double()
    rel = (40 + 8 * z) * E32
    fb.within(y[:, :7], a, rel * a.abs(), "y")
    # the derivative is a difference of two such terms, |a / g| and |d - a / g|
    f = (a / t).abs()
    fb.within(dx[:, :7], d, rel * (f + (d - a / t).abs()), "dx")
