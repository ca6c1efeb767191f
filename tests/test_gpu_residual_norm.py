"""residual_rms_norm and residual_rms_norm_fp8 against their plain form in 64 bits.

Bounds.  u = 2^-24 (fp32 half step), U = 2^-8 (bf16).  The mean square of D terms is summed in chains of at most D / 64 + 8
additions, so r has a relative error of at most (D / 64 + 16) u, y that and 4 roundings more, then the half step of its type.  A sum
over R rows (dweight) is off by (R + D / 64 + 24) u of the sizes of its terms; ds by the same of |w dy r| + |s| r^3 mean|w dy s|.
An e4m3 number is off by half a step, 2^-4 relative or 2^-10 of its smallest step, of the value that was rounded."""
import math

import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
u32, u16 = 2.0 ** -24, 2.0 ** -8


def step(t):
    return u16 if t == torch.bfloat16 else u32


def make(gen, shape, dt, rdt, res=True):
    x = torch.randn(*shape, generator=gen).to(dt)
    r = (3 * torch.randn(*shape, generator=gen)).to(rdt) if res else None
    return x, r, 0.5 + torch.rand(shape[-1], generator=gen)


@pytest.mark.parametrize("shape,dt,rdt", [((1, 1), torch.float32, torch.float32), ((3, 7), torch.bfloat16, torch.bfloat16),
                                          ((5, 64), torch.bfloat16, torch.float32), ((2, 3, 771), torch.float32, torch.float32),
                                          ((9, 1531), torch.bfloat16, torch.float32), ((4, 2048), torch.bfloat16, torch.bfloat16),
                                          ((3, 2049), torch.bfloat16, torch.bfloat16), ((2, 8192), torch.bfloat16, torch.float32),
                                          ((2, 16383), torch.float32, torch.float32), ((4099, 136), torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("res", [True, False])
def test_forward_and_gradients(gpu_device, shape, dt, rdt, res):
    gen = torch.Generator().manual_seed(sum(shape))
    x, r, w = make(gen, shape, dt, rdt, res)
    D, rows = shape[-1], math.prod(shape[:-1])
    from palimpsa_amd.ops.layer_glue import residual_rms_norm

    leaves = [None if t is None else t.to(gpu_device).requires_grad_(True) for t in (x, r, w)]
    y, s = residual_rms_norm(*leaves, eps=1e-5, residual_in_fp32=rdt == torch.float32)
    assert y.dtype == dt and s.dtype == rdt and y.shape == s.shape == x.shape
    ref = [None if t is None else t.double().requires_grad_(True) for t in (x, r, w)]
    yr, sr = bo.residual_norm(*ref, 1e-5, rdt)
    assert torch.equal(s.detach().cpu().double(), sr.detach().to(rdt).double())
    k = (D / 64 + 24) * u32
    assert ((y.detach().cpu().double() - yr.detach()).abs() <= (step(dt) + k) * yr.detach().abs() * 1.01).all()
    dy, ds = torch.randn(*shape, generator=gen).to(dt), torch.randn(*shape, generator=gen).to(rdt)
    have = [t for t in leaves if t is not None]
    got = torch.autograd.grad((y, s), have, (dy.to(gpu_device), ds.to(gpu_device)))
    want = torch.autograd.grad((yr, sr), [t for t in ref if t is not None], (dy.double(), ds.double()))
    sd, rr = sr.detach(), torch.rsqrt((sr.detach() ** 2).mean(-1, keepdim=True) + 1e-5)
    wd = (dy.double() * w.double()).abs()
    size = wd * rr + sd.abs() * rr ** 3 * (wd * sd.abs()).mean(-1, keepdim=True) + ds.double().abs()
    for g, v, t in zip(got[:-1], want, have):
        assert g.dtype == t.dtype
        assert ((g.cpu().double() - v).abs() <= step(t.dtype) * 1.01 * v.abs() + 2 * k * size).all()
    size = (dy.double() * sd * rr).abs().reshape(-1, D).sum(0)
    assert ((got[-1].cpu().double() - want[-1]).abs() <= (rows + D / 64 + 24) * u32 * size).all()


def test_one_gradient_alone_and_none(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm

    gen = torch.Generator().manual_seed(5)
    x, r, w = (t.to(gpu_device).requires_grad_(True) for t in make(gen, (6, 96), torch.float32, torch.float32))
    dy = torch.randn(6, 96, generator=gen).to(gpu_device)
    y, s = residual_rms_norm(x, r, w)
    both = torch.autograd.grad((y, s), (x, r, w), (dy, torch.zeros_like(s)), retain_graph=True)
    for a, b in zip(torch.autograd.grad(y, (x, r, w), dy, retain_graph=True), both):
        assert torch.equal(a, b)
    gx, gr, gw = torch.autograd.grad(s, (x, r, w), dy, allow_unused=True)
    assert torch.equal(gx, dy) and torch.equal(gr, dy) and not gw.any()


@pytest.mark.parametrize("D,group", [(8, None), (100, None), (96, 32), (2048, 128), (1536, 256), (4096, 64), (12288, None)])
@pytest.mark.parametrize("rdt", [torch.bfloat16, torch.float32])
def test_eight_bits(gpu_device, D, group, rdt):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm_fp8

    gen = torch.Generator().manual_seed(D)
    x, r, w = make(gen, (5, D), torch.bfloat16, rdt)
    x[2], r[2] = 0, 0                         # a row of nothing
    with torch.no_grad():
        q, sc, s = residual_rms_norm_fp8(x.to(gpu_device), r.to(gpu_device), w.to(gpu_device), group_size=group)
    y, sr = bo.residual_norm(x, r, w, 1e-5, rdt)
    g = group or D
    top = y.reshape(5, D // g, g).abs().amax(-1).clamp(min=1e-12)
    assert q.dtype == torch.float8_e4m3fn and tuple(sc.shape) == (5, D // g) and torch.equal(s.cpu().double(), sr)
    k = (D / 64 + 28) * u32
    assert ((sc.cpu().double() * 448 - top).abs() <= k * top).all()
    want = y.reshape(5, D // g, g) / (top / 448).unsqueeze(-1)
    have = q.cpu().float().double().reshape(want.shape)
    assert ((have - want).abs() <= (2.0 ** -4 + 2 * k) * want.abs() + 2.0 ** -10 * (1 + k)).all()
    assert have.abs().max() == 448


def test_eight_bits_of_rows_that_are_not_finite(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm, residual_rms_norm_fp8

    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(3)).to(gpu_device)
    x[1, 7], x[2, 200] = float("nan"), float("inf")
    q, sc, s = residual_rms_norm_fp8(x, None, torch.ones(256, device=gpu_device), group_size=128)
    assert torch.isnan(sc[1:3]).all() and torch.isfinite(sc[[0, 3]]).all() and torch.isfinite(q.float()[[0, 3]]).all()
    y, _ = residual_rms_norm(x, None, torch.ones(256, device=gpu_device))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 200]) and torch.isfinite(y[[0, 3]]).all()


def test_strides_and_types(gpu_device):
    """Slices of a wider projection, rows at odd addresses, parameters in bf16, fp16 rows (computed in fp32), an fp32 stream on demand."""
    from palimpsa_amd.ops.layer_glue import residual_rms_norm

    gen = torch.Generator().manual_seed(9)
    big = torch.randn(4, 6, 301, generator=gen).bfloat16().to(gpu_device)
    res = torch.randn(4, 6, 250, generator=gen).bfloat16().to(gpu_device)
    w = torch.rand(97, generator=gen).bfloat16().to(gpu_device)
    for x, r in ((big[..., 3:100], res[..., 1:98]), (big[:, ::2, 5:102], res[:, ::2, :97]), (big.transpose(0, 1)[..., :97], res.transpose(0, 1)[..., :97]),
                 (big[:1, :1, :97].expand(4, 6, 97), res[..., :97])):
        y, s = residual_rms_norm(x, r, w)
        yc, sc = residual_rms_norm(x.contiguous(), r.contiguous(), w)
        assert torch.equal(y, yc) and torch.equal(s, sc)
    y, s = residual_rms_norm(big[..., :97], None, w, residual_in_fp32=True)
    assert s.dtype == torch.float32 and torch.equal(s, big[..., :97].float())
    y16, s16 = residual_rms_norm(big[..., :97].half(), None, w)
    assert y16.dtype == torch.float16 and s16.dtype == torch.float32


def test_long_tensor(gpu_device):
    """Rows whose offsets pass 32 bits: the last rows equal those of a short call."""
    from palimpsa_amd.ops.layer_glue import residual_rms_norm

    rows, D = (1 << 31) // 1024 + 5, 1024
    x = torch.empty(rows, D, dtype=torch.bfloat16, device=gpu_device).fill_(0.5)
    x[-7:] = torch.randn(7, D, device=gpu_device).bfloat16()
    w = torch.ones(D, device=gpu_device)
    y, s = residual_rms_norm(x, x, w)
    ys, ss = residual_rms_norm(x[-7:], x[-7:], w)
    assert torch.equal(y[-7:], ys) and torch.equal(s[-7:], ss)
    assert torch.equal(y[0], y[rows // 2])


def test_refusals(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm, residual_rms_norm_fp8

    x, w = torch.randn(4, 96, device=gpu_device), torch.ones(96, device=gpu_device)
    for bad in (lambda: residual_rms_norm(x, x[:3], w), lambda: residual_rms_norm(x, x, w[:95]), lambda: residual_rms_norm(x[:0], None, w),
                lambda: residual_rms_norm(torch.empty(1, 16385, device=gpu_device), None, torch.ones(16385, device=gpu_device)),
                lambda: residual_rms_norm(x, x, w, eps=-1.0), lambda: residual_rms_norm(x, x.cpu(), w),
                lambda: residual_rms_norm_fp8(x, x, w, group_size=64), lambda: residual_rms_norm_fp8(x, x, w, group_size=48),
                lambda: residual_rms_norm_fp8(x.requires_grad_(True), x, w)):
        with pytest.raises(ValueError):
            bad()


def test_equal_calls_give_equal_bits_and_replay(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm

    gen = torch.Generator().manual_seed(4)
    x, r, w = (t.to(gpu_device).requires_grad_(True) for t in make(gen, (700, 520), torch.bfloat16, torch.float32))
    dy = torch.randn(700, 520, generator=gen).bfloat16().to(gpu_device)

    def pass_():
        y, s = residual_rms_norm(x, r, w)
        return (y.detach(), s.detach()) + torch.autograd.grad((y, s), (x, r, w), (dy, s.detach()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = pass_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pass_()
    for k in range(3):
        with torch.no_grad():
            x.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, pass_()):
            assert torch.equal(a, b), k
    with torch.no_grad():
        x.mul_(-1)
    for a, b in zip(first, pass_()):
        assert torch.equal(a, b)
