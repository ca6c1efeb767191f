"""Calls at the edges of the residual norm, the short convolution and the selective scan: few and many tokens in place, tensors that start
off a multiple of 16 bytes or lie far apart, broadcast inputs, one tensor in several places, captured training steps that share a pool.

Bounds: those of tests/test_gpu_selective_scan.py, k = (48 T + 64 + N + ch) half steps of fp32 of the sizes of the terms."""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
u32 = 2.0 ** -24


def inputs(gen, B, T, D, N):
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(u=r(B, T, D), delta=.5 * r(B, T, D), A=-torch.rand(D, N, generator=gen) - .01, B=r(B, T, N), C=r(B, T, N), D=r(D),
                z=r(B, T, D), delta_bias=.3 * r(D) - 1)


@pytest.mark.parametrize("N", [1, 4, 5, 8, 16, 24, 32, 64])
@pytest.mark.parametrize("B,T,D", [(1, 1, 9), (2, 3, 70), (3, 4, 130), (2, 5, 40), (1, 100, 40)])
def test_step_of_few_and_many_tokens_in_place(gpu_device, B, T, D, N):
    """Up to four tokens have a kernel of their own for some N; many tokens of few channels run in segments, and the state they start
    with is the place that the last of them writes."""
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step
    gen = torch.Generator().manual_seed(T * N)
    inp = inputs(gen, B, T, D, N)
    h0 = torch.randn(B, D, N, generator=gen)
    p = {n: t.to(gpu_device) for n, t in inp.items()}
    st = h0.to(gpu_device)
    with torch.no_grad():
        y = selective_scan_step(p.pop("u"), st, **p)
    (yr, fr, _, _), (ym, fm, _, _) = bo.scan(**inp, init=h0), bo.scan(**inp, init=h0, mass=True)
    k = (48 * T + 64 + N + D) * u32
    assert ((y.cpu().double() - yr).abs() <= k * ym).all() and ((st.cpu().double() - fr).abs() <= k * fm).all()
    y2, f2 = selective_scan(inp["u"].to(gpu_device), **p, initial_state=h0.to(gpu_device), output_final_state=True)
    assert torch.equal(y, y2) and torch.equal(st, f2)


def test_tensors_off_alignment_and_far_apart(gpu_device):
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step
    gen = torch.Generator().manual_seed(2)
    B, T, D, N = 2, 50, 40, 16
    inp = inputs(gen, B, T, D, N)
    h0, df = torch.randn(B, D, N, generator=gen), torch.randn(B, D, N, generator=gen)
    off = lambda t: torch.cat([torch.zeros(1), t.flatten()]).to(gpu_device)[1:].view(t.shape)  # noqa: E731
    leaves = []
    for place in (lambda t: t.to(gpu_device), off):
        p = {n: place(t).requires_grad_(True) for n, t in inp.items()}
        s = place(h0).requires_grad_(True)
        y, f = selective_scan(**p, initial_state=s, output_final_state=True)
        leaves.append([y, f, *torch.autograd.grad((y, f), [*p.values(), s], (torch.ones_like(y), place(df)))])
    assert off(h0).data_ptr() % 16 and all(torch.equal(a, b) for a, b in zip(*leaves))
    p = {n: t.to(gpu_device)[:, 0].contiguous() if n in ("u", "delta", "B", "C", "z") else t.to(gpu_device) for n, t in inp.items()}
    with pytest.raises(ValueError, match="16 bytes"):
        selective_scan_step(p.pop("u"), off(h0), **p)
    far = torch.zeros(3, 1 << 24, device=gpu_device)
    far[:, :D] = inp["u"][0, :3].to(gpu_device)
    x = far.as_strided((1, 3, D), (3 << 24, 1 << 24, 1))
    c = {n: t[:1, :3].to(gpu_device) if n in ("delta", "B", "C", "z") else t.to(gpu_device) for n, t in inp.items() if n != "u"}
    assert torch.equal(selective_scan(x, **c)[0], selective_scan(x.contiguous(), **c)[0])


def test_broadcast_and_repeated_inputs(gpu_device):
    """A row or a group that is expanded over the batch or the time gets the sum of what its copies get; so does a tensor that is three
    inputs at once."""
    from palimpsa_amd.ops.selective_scan import selective_scan
    gen = torch.Generator().manual_seed(5)
    B, T, D, N = 2, 20, 24, 16
    p = {n: t.to(gpu_device) for n, t in inputs(gen, B, T, D, N).items()}
    for name, shape in (("u", (1, 1, D)), ("B", (1, T, N)), ("C", (B, 1, N)), ("delta", (1, T, D))):
        small = torch.randn(shape, generator=gen).to(gpu_device).requires_grad_(True)
        whole = small.detach().expand(p[name].shape).clone().requires_grad_(True)
        out = []
        for t in (small.expand(p[name].shape), whole):
            y, _ = selective_scan(**{**p, name: t})
            out.append(torch.autograd.grad(y.square().sum(), small if t is not whole else whole)[0])
        dims = [d for d, s in enumerate(shape) if s != p[name].shape[d]]
        assert torch.allclose(out[0], out[1].sum(dims, keepdim=True), rtol=1e-5, atol=1e-4 * out[1].abs().max().item())
    t = torch.randn(B, T, D, generator=gen).to(gpu_device).requires_grad_(True)
    c = {n: x for n, x in p.items() if n not in ("u", "delta", "z")}
    g, = torch.autograd.grad(selective_scan(t, t, z=t, **c)[0].sum(), t)
    td = t.detach().cpu().double().requires_grad_(True)
    r, = torch.autograd.grad(bo.scan(td, td, z=td, **{n: x.cpu() for n, x in c.items()})[0].sum(), td)
    assert (g.cpu().double() - r).abs().max() <= 1e-4 * r.abs().max()


def test_gradient_of_one_output_alone(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm
    from palimpsa_amd.ops.selective_scan import selective_scan
    from palimpsa_amd.ops.short_conv import short_conv
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(2, 9, 24, generator=gen).to(gpu_device).requires_grad_(True)
    w = torch.randn(24, 4, generator=gen).to(gpu_device).requires_grad_(True)
    f = short_conv(x, w, output_final_state=True)[1]
    gx, gw = torch.autograd.grad(f.sum(), (x, w))          # the final state is the last four inputs
    assert gx[:, -4:].eq(1).all() and gx[:, :-4].eq(0).all() and gw.eq(0).all()
    n = torch.ones(24, device=gpu_device, requires_grad=True)
    s = residual_rms_norm(x, None, n)[1]
    gx, gn = torch.autograd.grad(s.sum(), (x, n))
    assert gx.eq(1).all() and gn.eq(0).all()
    p = {k: t.to(gpu_device) for k, t in inputs(gen, 2, 9, 24, 8).items()}
    p["C"].requires_grad_(True)
    f = selective_scan(**{**p, "u": x}, output_final_state=True)[1]
    gx, gc = torch.autograd.grad(f.sum(), (x, p["C"]))     # C and the gate come behind the state
    assert gc.eq(0).all() and gx.abs().max() > 0


def test_captured_training_steps_share_a_pool(gpu_device):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm
    from palimpsa_amd.ops.selective_scan import selective_scan
    from palimpsa_amd.ops.short_conv import short_conv
    gen = torch.Generator().manual_seed(8)
    p = {n: t.to(gpu_device) for n, t in inputs(gen, 2, 300, 40, 16).items()}
    x, w, n = (t.to(gpu_device).requires_grad_(True) for t in (p.pop("u"), torch.randn(40, 4, generator=gen), torch.ones(40)))
    A = p.pop("A").requires_grad_(True)

    def step():
        y, s = residual_rms_norm(x, None, n)
        o = selective_scan(short_conv(y, w)[0], p["delta"], A, p["B"], p["C"], z=p["z"])[0] + s
        return torch.autograd.grad(o.square().sum(), (x, w, n, A))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = step()
    with torch.cuda.graph(second, pool=first.pool()):
        b = step()
    for _ in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(2, 300, 40, generator=gen))
        first.replay()
        got = [t.clone() for t in a]
        second.replay()
        again = [t.clone() for t in b]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) and torch.equal(k, j) for i, j, k in zip(got, want, again))


def test_types_that_are_converted_and_refusals_with_gradients(gpu_device):
    """A call that is refused is refused before anything is launched, with gradients on as without."""
    from palimpsa_amd.ops.layer_glue import residual_rms_norm
    from palimpsa_amd.ops.selective_scan import selective_scan
    from palimpsa_amd.ops.short_conv import short_conv
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(2, 9, 24, generator=gen).to(gpu_device)
    w = torch.randn(24, 4, generator=gen).to(gpu_device).requires_grad_(True)
    y, _ = short_conv(x.half(), w)
    assert y.dtype == torch.float16 and torch.equal(y, short_conv(x.half().float(), w)[0].half())
    assert torch.autograd.grad(y.float().sum(), w)[0].dtype == torch.float32
    p = {n: t.to(gpu_device) for n, t in inputs(gen, 2, 9, 24, 8).items()}
    for bad in (lambda: short_conv(x, torch.randn(24, 9, device=gpu_device, requires_grad=True)),
                lambda: short_conv(x, torch.randn(24, 1, device=gpu_device, requires_grad=True)),
                lambda: short_conv(x, w[:-1]), lambda: short_conv(x[:, :0], w), lambda: short_conv(x[:0], w),
                lambda: short_conv(x, w, activation="relu"),
                lambda: selective_scan(**{**p, "A": torch.ones(24, 65, device=gpu_device, requires_grad=True)}),
                lambda: selective_scan(**{**p, "B": p["B"][:, :-1]}), lambda: selective_scan(**{**p, "C": p["C"].cpu()}),
                lambda: selective_scan(**{n: t[:, :0] if t.dim() == 3 else t for n, t in p.items()}),
                lambda: residual_rms_norm(torch.randn(2, 16385, device=gpu_device), None, torch.ones(16385, device=gpu_device, requires_grad=True)),
                lambda: residual_rms_norm(x, x[:1], torch.ones(24, device=gpu_device, requires_grad=True)),
                lambda: residual_rms_norm(x, None, torch.ones(24, device=gpu_device), float("nan"))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,G,ch", [(16, 1, 70), (40, 2, 140), (64, 1, 12), (3, 5, 35)])
def test_packs_of_ragged_sequences(gpu_device, N, G, ch, dt):
    """Sequences of 0 to 70 tokens, their starts and ends anywhere in blocks, segments and pairs of tokens, with states in and out and all
    gradients.  A term lives through its sequence's steps, at most 70 each way: k = (48 x 70 + 64 + N + ch) half steps."""
    from palimpsa_amd.ops.selective_scan import selective_scan
    gen = torch.Generator().manual_seed(N + ch)
    lens = torch.randint(0, 71, (18,), generator=gen).tolist() + [0, 1, 1, 2, 0, 7, 8, 9, 16, 64, 0]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T, S = cu[-1], len(lens)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    inp = dict(u=r(1, T, ch).to(dt), delta=(.5 * r(1, T, ch)).to(dt), A=-2 * torch.rand(ch, N, generator=gen), B=r(1, T, G, N).to(dt),
               C=r(1, T, G, N).to(dt), D=r(ch), z=r(1, T, ch).to(dt), delta_bias=.3 * r(ch) - 1)
    h0, dy, df = r(S, ch, N), r(1, T, ch).to(dt), r(S, ch, N)
    lv = {n: t.to(gpu_device).requires_grad_(True) for n, t in inp.items()}
    s0 = h0.to(gpu_device).requires_grad_(True)
    y, f = selective_scan(**lv, initial_state=s0, output_final_state=True, cu_seqlens=torch.tensor(cu, device=gpu_device))
    got = dict(zip([*("d" + n for n in lv), "d_init"], torch.autograd.grad((y, f), [*lv.values(), s0], (dy.to(gpu_device), df.to(gpu_device)))))
    kw = dict(**inp, init=h0, cu=cu)
    (yr, fr, _, _), (ym, fm, _, _) = bo.scan(**kw), bo.scan(**kw, mass=True)
    want, mass = bo.scan_grads(dy, d_final=df, **kw), bo.scan_grads(dy, d_final=df, **kw, mass=True)
    half = 2.0 ** -8 if dt == torch.bfloat16 else u32
    k = (48 * 70 + 64 + N + ch) * u32
    off = lambda t, ref: (t.detach().cpu().double() - ref).abs()  # noqa: E731
    assert (off(y, yr) <= 1.01 * half * yr.abs() + k * ym).all() and (off(f, fr) <= k * fm).all()
    for n, g in got.items():
        own = half if n in ("du", "ddelta", "dB", "dC", "dz") else u32
        chain = T if n in ("dA", "dD", "ddelta_bias") else 0
        assert (off(g, want[n]) <= 1.01 * own * want[n].abs() + (k + chain * u32) * mass[n]).all(), n


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 5, 8, 9, 15, 504, 513, 1027, 2047, 2055, 5000, 10001])
def test_norm_of_any_row_length(gpu_device, D, dt):
    """Rows whose last piece is moved back, of less than a piece, of lanes and waves without a piece; and nothing behind the last row.

    A lane adds at most 64 squares one after the other and the lanes 6 times more: r is off by 40 half steps, y by 64, dx by 128 of the
    sizes of its terms, dw by those and one for each row, every result by the half step of its type."""
    from palimpsa_amd.ops.layer_glue import residual_rms_norm, residual_rms_norm_fp8
    gen = torch.Generator().manual_seed(D)
    n = 5
    x, res, dy, ds = (torch.randn(n, D, generator=gen).to(dt) for _ in range(4))
    w = .5 + torch.rand(D, generator=gen)
    lv = [t.to(gpu_device).requires_grad_(True) for t in (x, res, w)]
    y, s = residual_rms_norm(*lv, 1e-5)
    gx, gr, gw = torch.autograd.grad((y, s), lv, (dy.to(gpu_device), ds.to(gpu_device)))
    half = 2.0 ** -8 if dt == torch.bfloat16 else u32
    sd = s.detach().cpu().double()
    assert ((sd - (x.double() + res.double())).abs() <= 1.01 * half * (x.double() + res.double()).abs()).all()
    r = torch.rsqrt((sd * sd).mean(-1, keepdim=True) + 1e-5)
    g, wd = dy.double(), w.double()
    c = lambda t: t.detach().cpu().double()  # noqa: E731
    yr = sd * r * wd
    assert ((c(y) - yr).abs() <= (1.01 * half + 64 * u32) * yr.abs()).all()
    dot, size = (g * wd * sd).sum(-1, keepdim=True), (g * wd * sd).abs().sum(-1, keepdim=True)
    dr = r * g * wd - sd * r ** 3 * dot / D + ds.double()
    mass = r * (g * wd).abs() + sd.abs() * r ** 3 * size / D + ds.double().abs()
    for t in (gx, gr):
        assert ((c(t) - dr).abs() <= 1.01 * half * dr.abs() + 128 * u32 * mass).all()
    dw, mw = (g * sd * r).sum(0), (g * sd * r).abs().sum(0)
    assert ((c(gw) - dw).abs() <= (64 + n) * u32 * mw).all()
    with torch.no_grad():
        q, scales, s8 = residual_rms_norm_fp8(lv[0], lv[1], lv[2], 1e-5)
    top = yr.abs().amax(-1, keepdim=True).clamp(min=1e-12) / 448
    assert torch.equal(s8, s) and ((c(scales) - top).abs() <= 70 * u32 * top).all()
    assert ((q.float().cpu().double() * c(scales) - yr).abs() <= 2.0 ** -4 * 1.01 * yr.abs() + 2.0 ** -10 * 1.01 * top).all()
