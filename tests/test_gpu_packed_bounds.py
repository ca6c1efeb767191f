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
