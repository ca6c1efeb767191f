"""selective_scan and selective_scan_step against their plain form in 64 bits.

Bounds.  u = 2^-24, U = 2^-8 (half steps of fp32 and bf16).  One step multiplies a state by exp(dt A), whose exponent is rounded twice (an
error of 3 u |dt A|, at most 12 u for the |dt A| <= 4 of these inputs; the time step itself is off by 8 u), and adds a product of
three: 24 u a step.  A term lives through at most T steps forward and T backward, and a sum over n, d or t adds one rounding for each addition in
a chain, so everything is off by at most k u = (48 T + 64 + chain) u of the sizes of its terms (the same formulas on absolute values)."""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
u32, u16 = 2.0 ** -24, 2.0 ** -8


def make(gen, bt, T, ch, N, G, dt, seqs=None, groups_dim=True):
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    bc = (bt, T, G, N) if groups_dim else (bt, T, N)
    inp = dict(u=r(bt, T, ch).to(dt), delta=(0.5 * r(bt, T, ch)).to(dt), A=-2 * torch.rand(ch, N, generator=gen), B=r(*bc).to(dt), C=r(*bc).to(dt),
               D=r(ch), z=r(bt, T, ch).to(dt), delta_bias=r(ch).clamp(-3, 0.5) - 1)
    return inp, None if seqs is None else r(seqs, ch, N)


CASES = [
    # bt, T, ch, N, G, dtype, softplus, state, cu, left out
    (1, 1, 1, 1, 1, torch.float32, True, True, None, ()),
    (2, 5, 3, 4, 1, torch.bfloat16, True, False, None, ("z",)),
    (1, 33, 70, 16, 1, torch.float32, True, True, None, ()),
    (2, 40, 64, 16, 1, torch.bfloat16, True, True, None, ()),
    (1, 21, 130, 5, 2, torch.float32, False, True, None, ("D",)),
    (1, 150, 24, 24, 2, torch.float32, True, False, None, ()),
    (1, 70, 20, 48, 1, torch.bfloat16, True, True, None, ("delta_bias",)),
    (1, 50, 12, 64, 4, torch.float32, True, True, None, ("D", "z", "delta_bias")),
    (1, 130, 17, 16, 1, torch.float32, True, True, [0, 0, 1, 3, 3, 20, 36, 64, 65, 130, 130], ()),
    (1, 200, 8, 20, 1, torch.bfloat16, True, False, [0, 64, 128, 130, 200], ()),
    (1, 260, 6, 33, 2, torch.float32, True, True, [0, 63, 63, 260], ()),
]


@pytest.mark.parametrize("bt,T,ch,N,G,dt,softplus,state,cu,without", CASES)
def test_forward_and_gradients(gpu_device, bt, T, ch, N, G, dt, softplus, state, cu, without):
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(T + ch)
    seqs = bt if cu is None else len(cu) - 1
    inp, s0 = make(gen, bt, T, ch, N, G, dt, seqs if state else None, groups_dim=G > 1 or T % 2 == 0)
    if not softplus:
        inp["delta"], inp["delta_bias"] = inp["delta"].abs(), inp["delta_bias"].abs() * 0.1
    for n in without:
        inp[n] = None
    dy, df = torch.randn(bt, T, ch, generator=gen).to(dt), torch.randn(seqs, ch, N, generator=gen)
    lv = {n: None if t is None else t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
    i0 = None if s0 is None else s0.to(gpu_device).requires_grad_(True)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=gpu_device)
    y, fin = selective_scan(**lv, delta_softplus=softplus, initial_state=i0, output_final_state=True, cu_seqlens=cut)
    names = [n for n in lv if lv[n] is not None] + (["init"] if state else [])
    leaves = [lv[n] for n in lv if lv[n] is not None] + ([i0] if state else [])
    got = dict(zip(names, torch.autograd.grad((y, fin), leaves, (dy.to(gpu_device), df.to(gpu_device)))))
    out = u16 if dt == torch.bfloat16 else u32
    kw = dict(**inp, softplus=softplus, init=s0, cu=cu)
    (yr, fr, _, _), (ym, fm, _, _) = bo.scan(**kw), bo.scan(**kw, mass=True)
    k = (48 * T + 64 + N + ch) * u32
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    assert ((d(y) - yr).abs() <= 1.01 * out * yr.abs() + k * ym).all()
    assert ((d(fin) - fr).abs() <= k * fm).all()
    want, mass = bo.scan_grads(dy, d_final=df, **kw), bo.scan_grads(dy, d_final=df, **kw, mass=True)
    for n in names:
        half = out if n in ("u", "delta", "B", "C", "z") else u32
        chain = bt * T if n in ("A", "D", "delta_bias") else 0
        off = (d(got[n]) - want["d_" + n if n == "init" else "d" + n]).abs()
        ref, m = (t["d_" + n if n == "init" else "d" + n] for t in (want, mass))
        bad = off > 1.01 * half * ref.abs() + (k + chain * u32) * m
        assert not bad.any(), (n, off.max(), ref.abs().max())


def test_a_gradient_is_a_difference(gpu_device):
    """The loss in fp32 on the GPU along a direction, a step of 2^-5 either way: the third derivative's share is below 1e-3 of it here, and
    rounding (1e-6 of the loss's terms over the step) below that."""
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(21)
    inp, s0 = make(gen, 1, 24, 20, 16, 1, torch.float32, 1)
    lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
    dy = torch.randn(1, 24, 20, generator=gen).to(gpu_device)
    g = dict(zip(lv, torch.autograd.grad(selective_scan(**lv, initial_state=s0.to(gpu_device))[0], list(lv.values()), dy)))
    for n in lv:
        v = torch.randn(lv[n].shape, generator=gen).to(gpu_device)
        v = v * 0.25 / v.abs().max()
        h = 2.0 ** -5
        f = lambda e: (selective_scan(**{**lv, n: lv[n] + e * v}, initial_state=s0.to(gpu_device))[0].double() * dy.double()).sum()  # noqa: E731
        with torch.no_grad():
            diff = (f(h) - f(-h)) / (2 * h)
        exact = (g[n].double() * v.double()).sum()
        size = (g[n].double() * v.double()).abs().sum()
        assert abs(diff - exact) <= 1e-3 * size, n


def test_pieces_equal_the_whole_and_steps_follow(gpu_device):
    """A prompt in two parts, then token by token and three at once.  Equal to the rounding of the parts' different orders; a step and a
    prompt of one token walk the same way: equal bits."""
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step

    gen = torch.Generator().manual_seed(13)
    inp, s0 = make(gen, 3, 40, 50, 16, 1, torch.float32, 3, groups_dim=False)
    p = {n: t.to(gpu_device) for n, t in inp.items()}
    cut = lambda a, b: {n: t[:, a:b] if n in ("u", "delta", "B", "C", "z") else t for n, t in p.items()}  # noqa: E731
    y, fin = selective_scan(**p, initial_state=s0.to(gpu_device), output_final_state=True)
    y1, st = selective_scan(**cut(0, 13), initial_state=s0.to(gpu_device), output_final_state=True)
    y2, st = selective_scan(**cut(13, 30), initial_state=st, output_final_state=True)
    parts = [y1, y2]
    for t in range(30, 34):
        one, nxt = selective_scan(**cut(t, t + 1), initial_state=st, output_final_state=True)
        v = st._version
        c = {n: x.squeeze(1) if n in ("u", "delta", "B", "C", "z") else x for n, x in cut(t, t + 1).items()}
        yt = selective_scan_step(c.pop("u"), st, **c)
        assert torch.equal(yt, one[:, 0]) and torch.equal(st, nxt) and st._version > v
        parts.append(yt.unsqueeze(1))
    for a, b in ((34, 37), (37, 40)):
        c = cut(a, b)
        parts.append(selective_scan_step(c.pop("u"), st, **c))
    kw = dict(**inp, init=s0)
    k = (48 * 40 + 200) * u32
    (_, _, _, _), (ym, fm, _, _) = bo.scan(**kw), bo.scan(**kw, mass=True)
    assert ((torch.cat(parts, 1) - y).abs().cpu().double() <= 2 * k * ym + 2 * u32 * ym).all()
    assert ((st - fin).abs().cpu().double() <= 2 * k * fm).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_long_sequences_in_segments(gpu_device, dt):
    """Few channels and many tokens run in segments; a pack of the same tokens with other channels beside them does not."""
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(17)
    T, ch, N = 3000, 40, 8
    inp, s0 = make(gen, 1, T, ch, N, 1, dt, 1)
    inp["A"] *= 0.1
    cu = [0, 700, 701, 701, 2500, T]
    init = torch.randn(5, ch, N, generator=gen)
    for bounds, st in ((None, s0), (cu, init)):
        lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
        i0 = st.to(gpu_device).requires_grad_(True)
        cut = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu_device)
        dy, df = torch.randn(1, T, ch, generator=gen).to(dt), torch.randn(st.shape, generator=gen)
        y, fin = selective_scan(**lv, initial_state=i0, output_final_state=True, cu_seqlens=cut)
        got = torch.autograd.grad((y, fin), list(lv.values()) + [i0], (dy.to(gpu_device), df.to(gpu_device)))
        kw = dict(**inp, init=st, cu=bounds)
        yr, fr, _, _ = bo.scan(**kw)
        want = bo.scan_grads(dy, d_final=df, **kw)
        out = u16 if dt == torch.bfloat16 else 1e-5     # fp32: relative to the largest, far below what T steps may give
        close = lambda a, r: ((a.detach().cpu().double() - r).abs() <= out * 1.01 * r.abs() + 2e-5 * r.abs().max()).all()  # noqa: E731
        assert close(y, yr) and close(fin, fr)
        for n, g in zip(list(lv) + ["_init"], got):
            assert close(g, want["d" + n]), n


def test_what_is_not_finite_stays_in_its_sequence(gpu_device):
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(19)
    inp, _ = make(gen, 1, 300, 20, 16, 1, torch.float32)
    p = {n: t.to(gpu_device) for n, t in inp.items()}
    p["u"][0, 70, 3], p["delta"][0, 130, 4] = float("nan"), float("inf")
    cu = torch.tensor([0, 64, 100, 131, 300], dtype=torch.int32, device=gpu_device)
    u = p["u"].clone().requires_grad_(True)
    y, f = selective_scan(**{**p, "u": u}, cu_seqlens=cu, output_final_state=True)
    bad = torch.isnan(y[0]).nonzero().tolist()
    assert {c for _, c in bad} == {3, 4} and min(t for t, c in bad if c == 3) == 70 and max(t for t, c in bad if c == 3) == 99
    assert torch.isfinite(f[[0, 3]]).all() and not torch.isfinite(f[1]).all()
    g, = torch.autograd.grad(y, u, torch.ones_like(y))
    assert torch.isfinite(g[0, 131:]).all() and torch.isfinite(g[0, :64]).all()


def test_extreme_inputs(gpu_device):
    """Time steps of zero, above the softplus' border and far below it, gates of +-200, decays that leave nothing."""
    from palimpsa_amd.ops.selective_scan import selective_scan

    gen = torch.Generator().manual_seed(23)
    inp, _ = make(gen, 1, 64, 64, 16, 1, torch.float32)
    inp["delta"][0, :8] = torch.linspace(-110, 60, 64)
    inp["delta_bias"].zero_()
    inp["z"][0, 8:16] = torch.linspace(-200, 200, 64)
    lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
    y, _ = selective_scan(**lv)
    dy = torch.randn(1, 64, 64, generator=gen)
    got = dict(zip(lv, torch.autograd.grad(y, list(lv.values()), dy.to(gpu_device))))
    yr, _, _, _ = bo.scan(**inp)
    ym, _, _, _ = bo.scan(**inp, mass=True)
    k = 1e-4      # exponents |dt A| up to 120: 3 u x 120 and what follows
    assert ((y.detach().cpu().double() - yr).abs() <= k * ym + 1e-30).all()
    want, mass = bo.scan_grads(dy, **inp), bo.scan_grads(dy, **inp, mass=True)
    for n in lv:
        assert ((got[n].cpu().double() - want["d" + n]).abs() <= k * mass["d" + n] + 1e-30).all(), n


def test_strides_and_types(gpu_device):
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step

    gen = torch.Generator().manual_seed(29)
    big = torch.randn(2, 60, 257, generator=gen).bfloat16().to(gpu_device)
    A, Dv = -torch.rand(33, 7, generator=gen).to(gpu_device), torch.randn(33, generator=gen).to(gpu_device)

    def views(t):
        return dict(u=t[..., 1:34], delta=t[..., 34:67], z=t[..., 70:103], B=t[..., 103:110], C=t[..., 111:118])

    for t in (big, big[:, ::2], big.transpose(0, 1)):
        v = views(t)
        c = {n: x.contiguous() for n, x in v.items()}
        l1, l2 = ({n: x.detach().requires_grad_(True) for n, x in d.items()} for d in (v, c))
        y1, f1 = selective_scan(**l1, A=A, D=Dv, output_final_state=True)
        y2, f2 = selective_scan(**l2, A=A, D=Dv, output_final_state=True)
        assert torch.equal(y1, y2) and torch.equal(f1, f2)
        for a, b in zip(torch.autograd.grad(y1, list(l1.values()), y1.detach()), torch.autograd.grad(y2, list(l2.values()), y2.detach())):
            assert torch.equal(a, b)
    v = {n: x[:, 5] for n, x in views(big).items()}
    s1 = torch.randn(2, 33, 7, generator=gen).to(gpu_device)
    s2 = s1.clone()
    with torch.no_grad():
        a = selective_scan_step(v["u"], s1, v["delta"], A, v["B"], v["C"], Dv, v["z"])
        b = selective_scan_step(*(t.contiguous() if i != 1 else t for i, t in enumerate((v["u"], s2, v["delta"], A, v["B"], v["C"], Dv, v["z"]))))
    assert torch.equal(a, b) and torch.equal(s1, s2)
    # one row of another type: everything in fp32, y in the type of u; a broadcast over the batch gets its gradient summed
    v = views(big)
    v["delta"] = v["delta"].float()
    assert selective_scan(**v, A=A.half())[0].dtype == torch.bfloat16
    one = big[:1, :, 103:110].detach().clone().requires_grad_(True)
    w = {**views(big), "B": one.expand(2, -1, -1)}
    g, = torch.autograd.grad(selective_scan(**w, A=A)[0], one, torch.ones(2, 60, 33, device=gpu_device).bfloat16())
    assert g.shape == one.shape


def test_long_tensor(gpu_device):
    """Offsets beyond 32 bits, forward and backward: the tail equals a short call that starts from the state, to the rounding of other segments."""
    from palimpsa_amd.ops.selective_scan import selective_scan

    T, ch, N = (1 << 31) // 1024 + 77, 1024, 2
    x = torch.empty(1, T, ch, dtype=torch.bfloat16, device=gpu_device).fill_(0.5)
    x[:, -300:] = torch.randn(1, 300, ch, device=gpu_device).bfloat16()
    bc = torch.randn(1, T, N, device=gpu_device).bfloat16()
    A = -torch.rand(ch, N, device=gpu_device) - 0.5
    x.requires_grad_(True)
    y, f = selective_scan(x, x.detach(), A, bc, bc, output_final_state=True)
    g, = torch.autograd.grad(y, x, x.detach())
    xs = x.detach()[:, -300:].clone().requires_grad_(True)
    ys, fs = selective_scan(xs, xs.detach(), A, bc[:, -300:], bc[:, -300:], output_final_state=True)
    gs, = torch.autograd.grad(ys, xs, xs.detach())
    # exp(-0.5 softplus(0.5)) is 0.61 a token: after 100 tokens nothing of what came before is left in fp32
    ok = lambda a, b: ((a.float() - b.float()).abs() <= 2 * u16 * b.float().abs() + 1e-5 * b.float().abs().max()).all()  # noqa: E731
    assert ok(y[:, -200:], ys[:, -200:]) and ok(f, fs) and ok(g[:, -200:], gs[:, -200:])


def test_refusals(gpu_device):
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step

    dev = gpu_device
    u, bc = torch.randn(2, 10, 6, device=dev), torch.randn(2, 10, 4, device=dev)
    A, st = -torch.rand(6, 4, device=dev), torch.zeros(2, 6, 4, device=dev)
    cu = torch.tensor([0, 5, 10], device=dev)
    ok = dict(u=u, delta=u, A=A, B=bc, C=bc)
    for kw in (dict(u=u[0]), dict(delta=u[:, :9]), dict(A=A[:5]), dict(A=A[0]), dict(B=bc[..., :3]), dict(C=bc[:, :9]), dict(D=A[:5, 0]), dict(z=u[..., :5]),
               dict(B=bc[0], C=bc[0]), dict(delta_bias=A[:, :1]), dict(initial_state=st[:1]), dict(cu_seqlens=cu),
               dict(A=-torch.rand(6, 65, device=dev), B=torch.randn(2, 10, 65, device=dev), C=torch.randn(2, 10, 65, device=dev)),
               dict(B=bc.unsqueeze(2).expand(2, 10, 4, 4), C=bc.unsqueeze(2).expand(2, 10, 4, 4)), dict(z=u.cpu()),
               dict(u=u[:, :0], delta=u[:, :0], B=bc[:, :0], C=bc[:, :0])):
        with pytest.raises(ValueError):
            selective_scan(**{**ok, **kw})
    one = (u[:, 0], st, u[:, 0], A, bc[:, 0], bc[:, 0])
    selective_scan_step(*one)
    for i, t in ((1, st[:1]), (1, st.bfloat16()), (1, st.transpose(1, 2).contiguous().transpose(1, 2)), (3, A.clone().requires_grad_(True)), (2, u)):
        with pytest.raises(ValueError):
            selective_scan_step(*(t if k == i else x for k, x in enumerate(one)))


def test_equal_bits_streams_and_replay(gpu_device):
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step

    gen = torch.Generator().manual_seed(31)
    inp, s0 = make(gen, 1, 700, 72, 16, 1, torch.bfloat16, 4)
    lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
    i0 = s0.to(gpu_device).requires_grad_(True)
    cu = torch.tensor([0, 100, 100, 333, 700], dtype=torch.int32, device=gpu_device)
    dy = torch.randn(1, 700, 72, generator=gen).bfloat16().to(gpu_device)

    def pass_():
        y, f = selective_scan(**lv, initial_state=i0, output_final_state=True, cu_seqlens=cu)
        return (y.detach(), f.detach()) + torch.autograd.grad((y, f), list(lv.values()) + [i0], (dy, f.detach()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = pass_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pass_()
    for k in range(4):
        with torch.no_grad():
            lv["u"].mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, pass_()):
            assert torch.equal(a, b), k
    for a, b in zip(first, pass_()):
        assert torch.equal(a, b)
    with torch.no_grad():
        c = {n: t.detach()[0, :4].clone() if n in ("u", "delta", "B", "C", "z") else t.detach() for n, t in lv.items()}
        u, st = c.pop("u"), i0.detach().clone()
        ref = st.clone()
        selective_scan_step(u, st, **c)
        st.copy_(ref)
        step = torch.cuda.CUDAGraph()
        with torch.cuda.graph(step):
            y = selective_scan_step(u, st, **c)
        for k in range(3):
            u.mul_(0.5)
            step.replay()
            want = selective_scan_step(u, ref, **c)
            assert torch.equal(y, want) and torch.equal(st, ref), k
