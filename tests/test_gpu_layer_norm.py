"""Layer norm and dropout on the GPU against their forms in 64 bits, forward and gradients, within the bounds of their roundings."""
import pytest
import torch

from oracle import feed_forward_oracle as fo
from tests import feed_forward_bounds as fb

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(dev, shape, dtype, res, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    D = shape[-1]
    out = dict(x=r(*shape).to(dtype), weight=r(D), bias=r(D), dy=r(*shape).to(dtype))
    out["residual"] = None if res is None else (2 * r(*shape) + 0.7).to(res)
    out["dres"] = None if res is None else r(*shape).to(res)
    return out


def dropped(t, p, seed, site):
    """Kept entries times the scale in fp32, in 64 bits."""
    keep = fo.kept(tuple(t.shape), p, seed, site).to(t.device)
    return torch.where(keep, t.double() * (1 / (1 - p)), 0.0)


SIZES = [1, 5, 8, 13, 64, 511, 512, 771, 1536, 2048, 2049, 4100, 8192, 16384]


@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_alone(gpu_device, D, dtype):
    from palimpsa_amd.ops.layer_glue import layer_norm
    for rows, bias in ((1, True), (9, False), (700 if D < 3000 else 40, True)):
        i = make(gpu_device, (rows, D), dtype, None, seed=D)
        b = i["bias"] if bias else None
        leaves = [t.clone().requires_grad_(True) for t in (i["x"], i["weight"], i["bias"])][:3 if bias else 2]
        y = layer_norm(*leaves, eps=1e-5)
        with torch.no_grad():
            assert torch.equal(y, layer_norm(i["x"], i["weight"], b, eps=1e-5))
        grads = torch.autograd.grad(y, leaves, i["dy"])
        val, tol = fb.layer_norm(i["x"], i["weight"], b, 1e-5, dtype, i["dy"])
        fb.within(y, val["y"], tol["y"], "y")
        fb.within(grads[0], val["ds"], tol["ds"] + fb.half_step(dtype) * val["ds"].abs(), "dx")
        fb.within(grads[1], val["weight"], tol["weight"], "dweight")
        if bias:
            fb.within(grads[2], val["bias"], tol["bias"], "dbias")


@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("dtype,res", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_of_the_stream(gpu_device, D, dtype, res, p):
    from palimpsa_amd.ops.layer_glue import residual_layer_norm
    shape, seed, site = (3, 7 if D > 3000 else 101, D), 0x123456789ABCDEF0 + D, 3
    i = make(gpu_device, shape, dtype, res, seed=D)
    leaves = {n: i[n].clone().requires_grad_(True) for n in ("x", "residual", "weight", "bias")}
    kw = dict(eps=1e-5, dropout_p=p, seed=seed, site=site)
    y, s = residual_layer_norm(**leaves, **kw)
    with torch.no_grad():
        y1, s1 = residual_layer_norm(**{n: t.detach() for n, t in leaves.items()}, **kw)
    assert torch.equal(y, y1) and torch.equal(s, s1) and y.dtype == dtype and s.dtype == res
    drop = lambda t: dropped(t, p, seed, site) if p else t.double()  # noqa: E731
    xs = drop(i["x"])
    want = xs + i["residual"].double()
    fb.within(s, want, fb.half_step(res) * want.abs() + 2 * fb.E32 * (xs.abs() + i["residual"].double().abs()), "s")
    val, tol = fb.layer_norm(s.detach(), i["weight"], i["bias"], 1e-5, dtype, i["dy"], i["dres"])
    fb.within(y, val["y"], tol["y"], "y")
    gx, gr, gw, gb = torch.autograd.grad([y, s], list(leaves.values()), [i["dy"], i["dres"]])
    fb.within(gr, val["ds"], tol["ds"] + fb.half_step(res) * val["ds"].abs(), "dresidual")
    dx, edx = drop(val["ds"]), drop(tol["ds"])
    fb.within(gx, dx, edx + (fb.half_step(dtype) + 2 * fb.E32) * dx.abs(), "dx")
    fb.within(gw, val["weight"], tol["weight"], "dweight")
    fb.within(gb, val["bias"], tol["bias"], "dbias")


def test_first_block_has_no_stream_yet(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_layer_norm
    i = make(gpu_device, (40, 776), BF, None)
    for fp32 in (False, True):
        x, w = i["x"].clone().requires_grad_(True), i["weight"].clone().requires_grad_(True)
        y, s = residual_layer_norm(x, None, w, residual_in_fp32=fp32, dropout_p=0.5, seed=9)
        assert s.dtype == (F32 if fp32 else BF)
        want = dropped(i["x"], 0.5, 9, 0)
        assert torch.equal(s.double(), want)               # a product by two is exact
        dres = torch.randn_like(s)
        gx, gw = torch.autograd.grad([y, s], [x, w], [i["dy"], dres])
        val, tol = fb.layer_norm(s.detach(), i["weight"], None, 1e-5, BF, i["dy"], dres)
        dx = dropped(val["ds"], 0.5, 9, 0)
        fb.within(gx, dx, dropped(tol["ds"], 0.5, 9, 0) + (2 ** -8 + 2 * fb.E32) * dx.abs(), "dx")
        fb.within(gw, val["weight"], tol["weight"], "dweight")
        # one of the two gradients alone
        (g1,) = torch.autograd.grad(residual_layer_norm(x, None, w, dropout_p=0.5, seed=9)[1].sum(), [x])
        assert torch.equal(g1.double(), dropped(torch.ones_like(x), 0.5, 9, 0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 1), (5, 3), (64, 8), (33, 100), (3, 1001, 771), (16, 768), (4097, 2048), (3, 70000)])
def test_dropout(gpu_device, dtype, shape):
    from palimpsa_amd.ops.layer_glue import dropout
    gen = torch.Generator(device=gpu_device).manual_seed(1)
    x = torch.randn(*shape, generator=gen, device=gpu_device).to(dtype)
    for p, seed, site in ((0.1, 1 << 40, 0), (0.75, -3, 0xFFFFFFFF)):
        leaf = x.clone().requires_grad_(True)
        y = dropout(leaf, p, seed, site)
        keep = fo.kept(shape, p, seed, site).to(gpu_device)
        want = torch.where(keep, x.float() * (1 / (1 - p)), 0.0).to(dtype)
        assert torch.equal(y, want)
        dy = torch.randn(*shape, generator=gen, device=gpu_device).to(dtype)
        (dx,) = torch.autograd.grad(y, [leaf], dy)
        assert torch.equal(dx, torch.where(keep, dy.float() * (1 / (1 - p)), 0.0).to(dtype))
    assert torch.equal(dropout(x, 0.0, 0), x)
