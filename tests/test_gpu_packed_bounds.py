"""Packed batches whose array of bounds was rewritten behind torch's back after it was checked: nothing outside the tensors is read.

States and rows stand inside larger buffers full of NaN, so that anything read beside them shows in the results."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def inside(t, dev):
    """t in the middle of a buffer of NaN, from a multiple of 16 bytes on."""
    n = t.numel()
    pad = 4096 + (-n) % 8
    big = torch.full((2 * pad + n,), float("nan"), dtype=t.dtype, device=dev)
    big[pad - pad % 8:][:n] = t.reshape(-1).to(dev)
    return big[pad - pad % 8:][:n].view(t.shape)


def rewrite(cu, values):
    cu.data.copy_(torch.tensor(values, dtype=torch.int32))     # (a view with a version of its own: the tensor does not count it)


@pytest.mark.parametrize("values", [[0, 10, 20, 20], [5, 20, 30, 60], [0, 10, 50, 60], [0, 60, 20, 10], [60, 60, 60, 60], [7, 7, 7, 7], [0, -5, 90, 30],
                                    [-(1 << 31), (1 << 31) - 1, -(1 << 31), 60]])
@pytest.mark.parametrize("N", [16, 20])
def test_scan(gpu_device, values, N):
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(5)
    T, ch = 60, 40
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    a = dict(u=r(1, T, ch), delta=r(1, T, ch), A=-torch.rand(ch, N, generator=gen), B=r(1, T, N), C=r(1, T, N), z=r(1, T, ch))
    lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in a.items()}
    init = inside(r(3, ch, N), gpu_device).requires_grad_(True)
    dy, df = inside(r(1, T, ch), gpu_device), inside(r(3, ch, N), gpu_device)
    cu = torch.tensor([0, 10, 30, 60], dtype=torch.int32, device=gpu_device)
    whole, _ = selective_scan(**lv, initial_state=init, cu_seqlens=cu)
    rewrite(cu, values)
    y, fin = selective_scan(**lv, initial_state=init, output_final_state=True, cu_seqlens=cu)
    got = torch.autograd.grad((y, fin), list(lv.values()), (dy, df))
    assert torch.isfinite(y).all()
    for n, g in zip(lv, got):
        assert torch.isfinite(g).all(), n
    rewrite(cu, [0, 10, 30, 60])
    again, _ = selective_scan(**lv, initial_state=init, cu_seqlens=cu)
    assert torch.equal(whole, again)


@pytest.mark.parametrize("W", [2, 4, 8])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("moved", [[0, 2, 40], [0, 0, 40], [0, 1, 3], [0, 40, 40], [0, 39, 3], [0, 50, 60], [-7, 2, 90]])
def test_convolution(gpu_device, W, dt, moved):
    """The table of tiles still is that of the bounds that were checked: a tile may start inside a sequence, fewer tokens from its start than
    the filter is long."""
    from palimpsa_amd.ops.short_conv import short_conv

    gen = torch.Generator().manual_seed(W)
    T, D = 40, 24
    x, dy = (inside(torch.randn(1, T, D, generator=gen).to(dt), gpu_device) for _ in range(2))
    x.requires_grad_(True)
    init, df = (inside(torch.randn(2, D, W, generator=gen).to(dt), gpu_device) for _ in range(2))
    init.requires_grad_(True)
    w, b = (torch.randn(*s, generator=gen).to(gpu_device).requires_grad_(True) for s in ((D, W), (D,)))
    cu = torch.tensor([0, 3, 40], dtype=torch.int32, device=gpu_device)
    whole, _ = short_conv(x, w, b, initial_state=init, cu_seqlens=cu)
    rewrite(cu, moved)
    y, fin = short_conv(x, w, b, initial_state=init, output_final_state=True, cu_seqlens=cu)
    gx, gw, gb = torch.autograd.grad((y, fin), (x, w, b), (dy, df))
    # rows that a tile of the old table and a sequence of the new bounds both hold are computed; the others are left as they are
    first, last = min(max(moved[1], 0), T), min(max(moved[2], 0), T)
    done = list(range(min(3, first))) + list(range(min(max(3, first), max(first, last)), max(first, last)))
    assert torch.isfinite(y[0, done]).all() and torch.isfinite(gx[0, done]).all() and torch.isfinite(fin).all()
    assert torch.isfinite(gw).all() and torch.isfinite(gb).all()
    rewrite(cu, [0, 3, 40])
    assert torch.equal(whole, short_conv(x, w, b, initial_state=init, cu_seqlens=cu)[0])
