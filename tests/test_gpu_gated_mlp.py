"""The gated feed-forward block on the GPU against its form in 64 bits, forward and gradients, within the bounds of its roundings."""
import pytest
import torch

from tests import feed_forward_bounds as fb

pytestmark = pytest.mark.gpu
NAMES = ("x", "w_gate", "w_up", "w_down")


def make(dev, M, D, F, Do, dtype, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    return [t.to(dtype) for t in (r(M, D), r(F, D) / D ** 0.5, r(F, D) / D ** 0.5, r(Do, F) / F ** 0.5)] + [r(M, Do).to(dtype)]


def check(dev, M, D, F, Do, dtype, act, seed=0):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    *inp, dy = make(dev, M, D, F, Do, dtype, seed)
    with torch.no_grad():
        plain = gated_mlp(*inp, activation=act)
    leaves = [t.clone().requires_grad_(True) for t in inp]
    y = gated_mlp(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    val, tol = fb.gated_mlp(*inp, act, dtype, dy)
    assert y.dtype == dtype and y.is_contiguous()
    assert torch.equal(y, plain), "with and without a gradient"
    fb.within(y, val["y"], tol["y"], "y")
    for n, g, t in zip(NAMES, grads, inp):
        assert g.shape == t.shape and g.dtype == t.dtype and g.is_contiguous()
        fb.within(g, val[n], tol[n], "d" + n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D,F,Do", [(1, 8, 8, 8), (3, 16, 24, 40), (16, 64, 136, 64), (17, 72, 200, 56), (33, 776, 520, 264), (64, 256, 96, 128),
                                      (65, 64, 128, 64), (100, 128, 256, 72), (128, 40, 64, 264), (257, 136, 328, 136), (300, 512, 640, 256),
                                      (1000, 96, 512, 96), (515, 768, 2048, 768)])
def test_against_the_form_in_64_bits(gpu_device, M, D, F, Do, dtype):
    print(M, D, F, Do, dtype, flush=True)
    check(gpu_device, M, D, F, Do, dtype, "silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [31, 32, 33, 48, 49, 64, 65])
@pytest.mark.parametrize("D,F,Do", [(256, 704, 256), (136, 4104, 72), (2048, 1408, 2048)])
def test_rows_about_the_kernels_of_few_rows(gpu_device, M, D, F, Do, dtype):
    check(gpu_device, M, D, F, Do, dtype, "silu")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [5, 130])
def test_activations(gpu_device, act, dtype, M):
    check(gpu_device, M, 96, 160, 96, dtype, act)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D,F,Do", [(1, 1, 1, 1), (7, 5, 3, 9), (70, 33, 65, 31), (129, 771, 1029, 385)])
def test_dims_that_are_no_multiple_of_eight(gpu_device, M, D, F, Do, dtype):
    check(gpu_device, M, D, F, Do, dtype, "silu")


@pytest.mark.parametrize("M,D,F", [(16384, 256, 512), (8192, 64, 4096), (2000, 2048, 1024)])
def test_many_rows(gpu_device, M, D, F):
    check(gpu_device, M, D, F, D, torch.bfloat16, "silu")
