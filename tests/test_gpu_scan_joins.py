"""The selective scan over so many segments that the waves of a join read theirs in several batches, with states that last through all of them.

5000 tokens of 40 channels are 157 segments of 32 tokens; a join's sixteen waves take ten each and read them eight at a time.  The decays are so
slow (dt |A| below 2e-3) that what a segment leaves is still there thousands of tokens later, and all factors have one sign, so that a segment
that is lost or counted twice moves what follows by 1 / 157 of it, a wave's run by ten times that.

Bounds.  u = 2^-24.  A step of a state is a decay off by at most 2 u (its exponent is so small that its roundings do not count) and one fused
operation: 3 u a step, and its input is off by 24 u.  So states, y and what comes back are off by (3 T + 24 + sums) u of the sizes of their terms, products of both
by twice that: (4 T + 200) u = 1.2e-3 forward and (8 T + 400) u = 2.4e-3 for gradients, of which 6.4e-3 is one segment."""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
u32, u16 = 2.0 ** -24, 2.0 ** -8


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cu", [None, [0, 37, 4400, 4400, 5000]])
def test_states_that_last(gpu_device, dt, cu):
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(41)
    T, ch, N = 5000, 40, 8
    seqs = 1 if cu is None else len(cu) - 1
    r = lambda *s: 0.1 + torch.rand(*s, generator=gen)  # noqa: E731
    inp = dict(u=r(1, T, ch).to(dt), delta=(r(1, T, ch) - 1).to(dt), A=-1e-3 * r(ch, N), B=r(1, T, N).to(dt), C=r(1, T, N).to(dt), D=r(ch),
               z=r(1, T, ch).to(dt), delta_bias=r(ch) - 1)
    init, dy, df = 500 * r(seqs, ch, N), r(1, T, ch).to(dt), 500 * r(seqs, ch, N)
    lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
    i0 = init.to(gpu_device).requires_grad_(True)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=gpu_device)
    y, fin = selective_scan(**lv, initial_state=i0, output_final_state=True, cu_seqlens=cut)
    got = torch.autograd.grad((y, fin), list(lv.values()) + [i0], (dy.to(gpu_device), df.to(gpu_device)))
    kw = dict(**inp, init=init, cu=cu)
    yr, fr, _, _ = bo.scan(**kw)
    want, mass = bo.scan_grads(dy, d_final=df, **kw), bo.scan_grads(dy, d_final=df, **kw, mass=True)
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    out = u16 if dt == torch.bfloat16 else u32
    k = (4 * T + 200) * u32
    assert ((d(y) - yr).abs() <= (1.01 * out + k) * yr).all() and ((d(fin) - fr).abs() <= (u32 + k) * fr).all()
    for n, g in zip(list(lv) + ["_init"], got):
        half = out if n in ("u", "delta", "B", "C", "z") else u32
        w, m = want["d" + n], mass["d" + n]
        assert ((d(g) - w).abs() <= 1.01 * half * w.abs() + (8 * T + 400) * u32 * m).all(), n
