"""short_conv and short_conv_step against their plain form in 64 bits.

Bounds.  u = 2^-24, U = 2^-8 (half steps of fp32 and bf16).  p is W + 1 fused operations: off by (W + 1) u of m = |bias| + sum |w x|; the
logistic function is off by 12 u and by its slope (at most 1/4 of p's error), so y is off by (W + 16) u (|y| + 1.1 m) and the half step
of its type.  The gradients are sums of products of dy, act' (a few u), w and x: off by (number of terms + 40) u of the sizes of the terms."""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
u32, u16 = 2.0 ** -24, 2.0 ** -8


def make(gen, B, T, D, W, dt, seqs=None):
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return r(B, T, D).to(dt), r(D, W) / W ** 0.5, r(D), None if seqs is None else r(seqs, D, W).to(dt)


CASES = [
    # B, T, D, W, dtype, silu, bias, state, cu
    (1, 1, 1, 2, torch.float32, True, True, True, None),
    (2, 3, 5, 4, torch.bfloat16, True, True, True, None),
    (2, 65, 8, 4, torch.bfloat16, False, False, False, None),
    (3, 64, 24, 3, torch.float32, True, True, True, None),
    (1, 200, 515, 4, torch.bfloat16, True, True, False, None),
    (1, 37, 130, 8, torch.float32, True, False, True, None),
    (2, 100, 64, 5, torch.bfloat16, True, True, True, None),
    (1, 150, 72, 4, torch.bfloat16, True, True, True, [0, 0, 1, 3, 3, 67, 131, 132, 150, 150]),
    (1, 90, 33, 4, torch.float32, False, True, False, [0, 2, 64, 65, 90]),
    (1, 77, 16, 7, torch.float32, True, True, True, [0, 3, 9, 9, 77]),
]


@pytest.mark.parametrize("B,T,D,W,dt,silu,bias,state,cu", CASES)
def test_forward_and_gradients(gpu_device, B, T, D, W, dt, silu, bias, state, cu):
    from palimpsa_amd.ops.short_conv import short_conv

    gen = torch.Generator().manual_seed(T + D)
    seqs = B if cu is None else len(cu) - 1
    x, w, b, s0 = make(gen, B, T, D, W, dt, seqs if state else None)
    b = b if bias else None
    dy, df = torch.randn(B, T, D, generator=gen).to(dt), torch.randn(seqs, D, W, generator=gen).to(dt)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=gpu_device)
    names = [n for n, t in (("x", x), ("w", w), ("b", b), ("s0", s0)) if t is not None]
    have = [t for t in (x, w, b, s0) if t is not None]

    def both(kind):
        lv = {n: (t.to(gpu_device) if kind else t.double()).detach().requires_grad_(True) for n, t in zip(names, have)}
        if kind:
            y, fin = short_conv(lv["x"], lv["w"], lv.get("b"), "silu" if silu else None, lv.get("s0"), True, cut)
            g = torch.autograd.grad((y, fin), list(lv.values()), (dy.to(gpu_device), df.to(gpu_device)))
        else:
            y, fin = bo.conv(lv["x"], lv["w"], lv.get("b"), silu, lv.get("s0"), cu)
            g = torch.autograd.grad((y, fin), list(lv.values()), (dy.double(), df.double()))
        return [t.detach().cpu().double() for t in (y, fin) + g]

    got, want = both(True), both(False)
    out = u16 if dt == torch.bfloat16 else u32
    ax = [None if t is None else t.double().abs() for t in (x, w, b, s0)]
    m = bo.conv(ax[0], ax[1], ax[2], False, ax[3], cu)[0]
    assert ((got[0] - want[0]).abs() <= 1.01 * out * want[0].abs() + (W + 16) * u32 * (want[0].abs() + 1.1 * m)).all()
    assert torch.equal(got[1], want[1])
    # sizes of the gradients' terms: the same differentiation of the bare convolution of absolute values, |act'| <= 1.1, and
    # act' moves by half of p's error
    lv = [t.detach().requires_grad_(True) for t in ax if t is not None]
    mass = bo.conv(lv[0], lv[1], lv[2] if bias else None, False, lv[-1] if state else None, cu)
    wts = (dy.double().abs() * (1.1 + m), df.double().abs())
    sizes = torch.autograd.grad(mass, lv, wts)
    terms = {"x": W + 1, "w": B * T, "b": B * T, "s0": W + 1}
    for n, g, v, z in zip(names, got[2:], want[2:], sizes):
        half = out if n in ("x", "s0") else u32
        assert ((g - v).abs() <= 1.01 * half * v.abs() + (terms[n] + W + 40) * u32 * z).all(), n


def test_pieces_equal_the_whole_and_steps_follow(gpu_device):
    """A prompt in two parts, then token by token and three tokens at once: the bits of one pass (fp32 and bf16)."""
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step

    for dt in (torch.float32, torch.bfloat16):
        gen = torch.Generator().manual_seed(7)
        x, w, b, s0 = (t.to(gpu_device) for t in make(gen, 3, 40, 44, 4, dt, 3))
        y, fin = short_conv(x, w, b, initial_state=s0, output_final_state=True)
        y1, st = short_conv(x[:, :13], w, b, initial_state=s0, output_final_state=True)
        y2, st = short_conv(x[:, 13:30], w, b, initial_state=st, output_final_state=True)
        parts = [y1, y2]
        for t in range(30, 34):
            v = st._version
            parts.append(short_conv_step(x[:, t], st, w, b).unsqueeze(1))
            assert st._version > v
        parts += [short_conv_step(x[:, 34:37], st, w, b), short_conv_step(x[:, 37:], st, w, b)]
        assert torch.equal(torch.cat(parts, 1), y) and torch.equal(st, fin)


def test_strides_and_types(gpu_device):
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step

    gen = torch.Generator().manual_seed(8)
    big = torch.randn(3, 50, 301, generator=gen).bfloat16().to(gpu_device)
    w = torch.randn(97, 1, 4, generator=gen).bfloat16().to(gpu_device)
    b = torch.randn(97, generator=gen).bfloat16().to(gpu_device)
    for x in (big[..., 3:100], big[:, ::2, 5:102], big[:1, :, :97].expand(3, 50, 97), big.transpose(0, 1)[..., 7:104], big[:, :1, 1:98],
              big[:, :, 0:194:2]):
        xr = x.clone().contiguous()
        for t in (x, xr):
            t = t.detach()
        y, f = short_conv(x, w, b, output_final_state=True)
        yc, fc = short_conv(xr, w, b, output_final_state=True)
        assert torch.equal(y, yc) and torch.equal(f, fc)
        l1, l2 = x.detach().requires_grad_(True), xr.detach().requires_grad_(True)
        g1, = torch.autograd.grad(short_conv(l1, w, b)[0], l1, y)
        g2, = torch.autograd.grad(short_conv(l2, w, b)[0], l2, y)
        assert torch.equal(g1, g2)
    s1 = torch.zeros(3, 97, 4, dtype=torch.bfloat16, device=gpu_device)
    s2 = s1.clone()
    with torch.no_grad():
        assert torch.equal(short_conv_step(big[:, 4, 9:106], s1, w, b), short_conv_step(big[:, 4, 9:106].contiguous(), s2, w, b))
    y16, f16 = short_conv(big[..., :97].half(), w.half(), b, output_final_state=True)
    assert y16.dtype == f16.dtype == torch.float16
    i64 = torch.tensor([0, 20, 50], device=gpu_device)
    assert torch.equal(short_conv(big[:1, :, :97], w, b, cu_seqlens=i64)[0], short_conv(big[:1, :, :97], w, b, cu_seqlens=i64.int())[0])


def test_what_is_not_finite_stays_in_its_sequence(gpu_device):
    from palimpsa_amd.ops.short_conv import short_conv

    x = torch.randn(1, 30, 16, device=gpu_device)
    x[0, 9, 3], x[0, 12, 5] = float("nan"), float("inf")
    cu = torch.tensor([0, 10, 30], dtype=torch.int32, device=gpu_device)
    w = torch.randn(16, 3, device=gpu_device)
    y, _ = short_conv(x, w, activation=None, cu_seqlens=cu)
    bad = ~torch.isfinite(y[0])
    assert bad.nonzero().tolist() == [[9, 3], [12, 5], [13, 5], [14, 5]]


def test_long_tensor(gpu_device):
    """Offsets beyond 32 bits, forward and backward: the tail equals that of a short call that starts from the state."""
    from palimpsa_amd.ops.short_conv import short_conv

    T, D = (1 << 31) // 1024 + 321, 1024
    x = torch.empty(1, T, D, dtype=torch.bfloat16, device=gpu_device).fill_(0.25)
    x[:, -200:] = torch.randn(1, 200, D, device=gpu_device).bfloat16()
    w, b = torch.randn(D, 4, device=gpu_device), torch.randn(D, device=gpu_device)
    xs = x[:, -200:].clone().requires_grad_(True)
    state = x[:, -204:-200].transpose(1, 2).contiguous()
    x.requires_grad_(True)
    y, f = short_conv(x, w, b, output_final_state=True)
    ys, fs = short_conv(xs, w, b, initial_state=state, output_final_state=True)
    assert torch.equal(y[:, -200:], ys) and torch.equal(f, fs)
    g, = torch.autograd.grad(y, x, y.detach())
    gs, = torch.autograd.grad(ys, xs, ys.detach())
    assert torch.equal(g[:, -200:], gs)


def test_refusals(gpu_device):
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step

    x, w = torch.randn(2, 10, 6, device=gpu_device), torch.randn(6, 4, device=gpu_device)
    st = torch.zeros(2, 6, 4, device=gpu_device)
    cu = torch.tensor([0, 5, 10], device=gpu_device)
    for bad in (lambda: short_conv(x[0], w), lambda: short_conv(x, w[:5]), lambda: short_conv(x, w[:, :1]), lambda: short_conv(x, w.repeat(1, 3)),
                lambda: short_conv(x, w, activation="gelu"), lambda: short_conv(x, w, w[:5, 0]), lambda: short_conv(x, w, initial_state=st[:1]),
                lambda: short_conv(x, w, cu_seqlens=cu), lambda: short_conv(x[:1], w, cu_seqlens=cu[:2]), lambda: short_conv(x[:, :0], w),
                lambda: short_conv(x, w.cpu()), lambda: short_conv_step(x[:, 0], st[:1], w), lambda: short_conv_step(x[:, 0], st.bfloat16(), w),
                lambda: short_conv_step(x[:, 0], st.transpose(0, 1), w), lambda: short_conv_step(x[:, 0], st, w.requires_grad_(True)),
                lambda: short_conv_step(x[:, 0].half(), st.half(), w.detach())):
        with pytest.raises(ValueError):
            bad()


def test_equal_bits_streams_and_replay(gpu_device):
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step

    gen = torch.Generator().manual_seed(11)
    x, w, b, s0 = (t.to(gpu_device).requires_grad_(True) for t in make(gen, 1, 600, 200, 4, torch.bfloat16, 3))
    cu = torch.tensor([0, 100, 101, 600], dtype=torch.int32, device=gpu_device)
    dy = torch.randn(1, 600, 200, generator=gen).bfloat16().to(gpu_device)

    def pass_():
        y, f = short_conv(x, w, b, initial_state=s0, output_final_state=True, cu_seqlens=cu)
        return (y.detach(), f.detach()) + torch.autograd.grad((y, f), (x, w, b, s0), (dy, f.detach()))

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
            x.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, pass_()):
            assert torch.equal(a, c), k
    for a, c in zip(first, pass_()):
        assert torch.equal(a, c)
    st, row = s0.detach().clone(), x.detach()[0, :3].clone()
    with torch.no_grad():
        ref, sr = st.clone(), []
        step = torch.cuda.CUDAGraph()
        short_conv_step(row, st, w, b)
        st.copy_(ref)
        with torch.cuda.graph(step):
            y = short_conv_step(row, st, w, b)
        for k in range(3):
            row.mul_(0.5)
            step.replay()
            want = short_conv_step(row, ref, w, b)
            assert torch.equal(y, want) and torch.equal(st, ref), k
