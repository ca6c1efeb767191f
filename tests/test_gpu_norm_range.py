"""residual_rms_norm where a workgroup's four waves walk several rows, and for rows of very small and very large entries.

Bounds as in test_gpu_residual_norm.py: u = 2^-24, U = 2^-8; r is off by (D / 64 + 16) u, y by that and 4 roundings, ds by (D / 64 + 24) u of
twice the sizes of its terms, dweight by (rows + D / 64 + 24) u of its, all behind the half step of the result's type; an 8-bit number by
2^-4 of the value that was rounded, or 2^-10."""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
u32, u16 = 2.0 ** -24, 2.0 ** -8


def check(dev, x, r, w, dy, ds, eps, rdt):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm

    rows, D = x.shape
    step = lambda t: u16 if t == torch.bfloat16 else u32  # noqa: E731
    have = [t for t in (x, r, w) if t is not None]
    lv = [t.to(dev).requires_grad_(True) for t in have]
    y, s = residual_rms_norm(lv[0], lv[1] if r is not None else None, lv[-1], eps, rdt == torch.float32)
    out, cot = ((y, s), (dy, ds)) if ds is not None else ((y,), (dy,))
    got = torch.autograd.grad(out, lv, [t.to(dev) for t in cot])
    ref = [t.double().requires_grad_(True) for t in have]
    yr, sr = bo.residual_norm(ref[0], ref[1] if r is not None else None, ref[-1], eps, rdt)
    want = torch.autograd.grad((yr, sr)[:len(cot)], ref, [t.double() for t in cot])
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    k = (D / 64 + 24) * u32
    yr, sr = yr.detach(), sr.detach()
    assert ((d(y) - yr).abs() <= (step(x.dtype) + k) * yr.abs() * 1.01).all()
    rr = torch.rsqrt((sr * sr).mean(-1, keepdim=True) + eps)
    wd, hat = (dy.double() * w.double()).abs(), sr.abs() * rr
    size = wd * rr + rr * hat * (wd * hat).mean(-1, keepdim=True) + (0 if ds is None else ds.double().abs())
    for g, v, t in zip(got[:-1], want, have):
        assert ((d(g) - v).abs() <= step(t.dtype) * 1.01 * v.abs() + 2 * k * size).all()
    assert ((d(got[-1]) - want[-1]).abs() <= (rows + D / 64 + 24) * u32 * (dy.double().abs() * hat).sum(0)).all()


@pytest.mark.parametrize("D,dt,rdt", [(2049, torch.bfloat16, torch.float32), (4096, torch.bfloat16, torch.bfloat16), (5000, torch.float32, torch.float32)])
def test_many_rows_of_four_waves(gpu_device, D, dt, rdt):
    """4500 rows: three rounds of the forward's 2048 workgroups, nine of the backward's 512."""
    gen = torch.Generator().manual_seed(D)
    n = lambda t: torch.randn(4500, D, generator=gen).to(t)  # noqa: E731
    check(gpu_device, n(dt), n(rdt), 0.5 + torch.rand(D, generator=gen), n(dt), n(rdt), 1e-5, rdt)


@pytest.mark.parametrize("D,group", [(2049, None), (4096, None), (4096, 256)])
def test_many_rows_of_four_waves_in_eight_bits(gpu_device, D, group):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm_fp8

    gen = torch.Generator().manual_seed(D)
    x = torch.randn(4500, D, generator=gen).bfloat16() * torch.exp(torch.randn(4500, 1, generator=gen)).bfloat16()
    w = 0.5 + torch.rand(D, generator=gen)
    q, sc, _ = residual_rms_norm_fp8(x.to(gpu_device), None, w.to(gpu_device), group_size=group)
    y, _ = bo.residual_norm(x, None, w, 1e-5, torch.bfloat16)
    y = y.reshape(4500, -1, group or D)
    top = y.abs().amax(-1)
    k = (D / 64 + 28) * u32
    assert ((sc.cpu().double() * 448 - top).abs() <= k * top).all()
    want = y * 448 / top.unsqueeze(-1)
    have = q.cpu().float().double().reshape(want.shape)
    assert ((have - want).abs() <= (2.0 ** -4 + 2 * k) * want.abs() + 2.0 ** -10 * (1 + k)).all()


@pytest.mark.parametrize("size,eps", [(1e-15, 0.0), (1e-13, 0.0), (1e12, 1e-5), (1e15, 1e-5), (1e17, 1e-5)])
@pytest.mark.parametrize("D,dt", [(5, torch.float32), (200, torch.float32), (200, torch.bfloat16), (2100, torch.float32)])
def test_sizes_of_rows(gpu_device, size, eps, D, dt):
    """The cube of 1 / rms passes the range of fp32 from 1e13 and 1e-13 on; the gradients, of size 1 / rms, do not."""
    gen = torch.Generator().manual_seed(D)
    n = lambda: torch.randn(9, D, generator=gen)  # noqa: E731
    check(gpu_device, (n() * size).to(dt), None, 0.5 + torch.rand(D, generator=gen), n().to(dt), None, eps, dt)
