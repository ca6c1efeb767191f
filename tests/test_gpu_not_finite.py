"""Infinities through the selective scan: every result is of the kind (finite, +inf, -inf, not a number) that the formulas give in 64 bits.

All factors have one sign (u, B, C, D, z, dy and the states positive, A negative), so that no sum has infinities of both signs in it and the kind
of a result does not hang on an order of sums; no product overflows by itself."""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
INF = float("inf")


def inputs(T, ch, N, G, dt, gate):
    gen = torch.Generator().manual_seed(100 * N + ch)
    r = lambda *s: (0.1 + torch.rand(*s, generator=gen))  # noqa: E731
    inp = dict(u=r(1, T, ch).to(dt), delta=r(1, T, ch).to(dt), A=-r(ch, N), B=r(1, T, G, N).to(dt), C=r(1, T, G, N).to(dt), D=r(ch),
               z=r(1, T, ch).to(dt) if gate else None, delta_bias=0.1 * r(ch))
    return inp, r(1, ch, N), r(1, T, ch).to(dt), r(1, ch, N)


def kind(t):
    t = t.detach().cpu().double()
    return torch.where(torch.isnan(t), 3.0, torch.where(torch.isinf(t), torch.sign(t), 2.0))


def check(dev, inp, init, dy, d_final, cu=None):
    from palimpsa_amd.ops.selective_scan import selective_scan

    lv = {n: None if t is None else t.to(dev).requires_grad_(True) for n, t in inp.items()}
    i0 = init.to(dev).requires_grad_(True)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    y, fin = selective_scan(**lv, initial_state=i0, output_final_state=True, cu_seqlens=cut)
    names = [n for n in lv if lv[n] is not None]
    got = torch.autograd.grad((y, fin), [lv[n] for n in names] + [i0], (dy.to(dev), d_final.to(dev)))
    kw = dict(**inp, init=init, cu=cu)
    yr, fr, _, _ = bo.scan(**kw)
    want = bo.scan_grads(dy, d_final=d_final, **kw)
    with torch.no_grad():
        plain, _ = selective_scan(**{n: None if t is None else t.detach() for n, t in lv.items()}, initial_state=i0, cu_seqlens=cut)
    assert torch.equal(kind(y), kind(yr)) and torch.equal(kind(plain), kind(yr)) and torch.equal(kind(fin), kind(fr))
    for n, g in zip(names + ["_init"], got):
        assert torch.equal(kind(g), kind(want["d" + n])), n
    assert (kind(yr) == 1).any()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,ch,G", [(1, 3, 1), (5, 70, 1), (8, 64, 1), (16, 64, 1), (20, 6, 2), (24, 64, 1), (40, 5, 1), (63, 64, 1)])
@pytest.mark.parametrize("gate", [True, False])
def test_an_infinite_input_or_time_step(gpu_device, N, ch, G, dt, gate):
    inp, init, dy, df = inputs(45, ch, N, G, dt, gate)
    inp["u"][0, 11, 0], inp["u"][0, 33, 1], inp["delta"][0, 19, 2] = INF, INF, INF
    check(gpu_device, inp, init, dy, df)


@pytest.mark.parametrize("N,ch", [(8, 3), (16, 64), (24, 70)])
def test_an_infinite_gradient(gpu_device, N, ch):
    inp, init, dy, df = inputs(45, ch, N, 1, torch.float32, True)
    inp["u"][0, 40, 1] = INF
    dy[0, 21, 0] = INF
    check(gpu_device, inp, init, dy, df)


@pytest.mark.parametrize("N,ch", [(3, 3), (16, 70), (24, 5)])
@pytest.mark.parametrize("where", ["init", "d_final", "delta_bias"])
def test_the_last_channel_of_a_tile(gpu_device, N, ch, where):
    """Lanes without a channel have nothing of the last channel's: sums over the channels (dB, dC) stay as they are."""
    inp, init, dy, df = inputs(45, ch, N, 1, torch.float32, True)
    inp["u"][0, 3, 0] = INF
    {"init": init, "d_final": df, "delta_bias": inp["delta_bias"].view(1, ch)}[where][0, -1] = INF
    check(gpu_device, inp, init, dy, df)


def test_through_many_segments(gpu_device):
    """3000 tokens of few channels run in 94 segments; the decay over a run of them is zero in fp32, and an infinite state stays infinite."""
    inp, init, dy, df = inputs(3000, 40, 1, 1, torch.float32, False)
    inp["u"][0, 5, 3], df[0, 7, 0] = INF, INF
    check(gpu_device, inp, init, dy, df)
    init, df = init.repeat(3, 1, 1), df.repeat(3, 1, 1)
    df[1] = 1.0
    check(gpu_device, inp, init, dy, df, [0, 1000, 1003, 3000])
