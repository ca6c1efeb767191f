"""The operators as a block strings them together: residual norm -> short convolution -> selective scan, and the convolution in front of
the recurrence of the framework; prompts, single tokens, gradients, packed batches and replayed graphs.

Bounds.  In fp32 a chain is off by the sum of what its links are off by, each amplified by the links behind it.  The values here are of
size one, a link's own error is below 64 half steps of the sizes of its terms (the bounds of the links' own tests), and what a link
amplifies is below 16 (norm: |w| / rms; convolution: sum |w| ~ 2; scan: 1 / (1 - a) <= 1 / (1 - e^-0.1 dt) over the length that counts);
two links behind the first: 64 * 16 * 16 half steps = 1e-3 of the largest value, for gradients, whose chains are twice as long, of the
largest gradient.  A lost token, state or term moves the results by far more than that."""
import pytest
import torch

from oracle import block_oracle as bo
from oracle import palimpsa_oracle as po

pytestmark = pytest.mark.gpu


def block_inputs(gen, B, T, D, N, W, S):
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(x=r(B, T, D), residual=r(B, T, D), wn=1 + .1 * r(D), wp=r(D, 3 * D + 2 * N) / D ** .5, wc=r(D, W) / W ** .5, bc=.1 * r(D),
                A=-torch.rand(D, N, generator=gen) - .1, Dp=r(D), bias=r(D) * .1, conv0=r(S, D, W), h0=r(S, D, N))


def block(a, D, N, cu, ops):
    norm, conv, scan = ops
    y, res = norm(a["x"], a["residual"], a["wn"])
    p = y @ a["wp"]
    xs, z, dl, B, C = p.split([D, D, D, N, N], -1)
    c, cf = conv(xs, a["wc"], a["bc"], a["conv0"])
    o, hf = scan(c, dl, a["A"], B, C, a["Dp"], z, a["bias"], a["h0"])
    return o + res, cf, hf


@pytest.mark.parametrize("B,T,cu", [(2, 70, None), (1, 1, None), (1, 83, [0, 0, 40, 41, 83])])
def test_block_with_gradients(gpu_device, B, T, cu):
    from palimpsa_amd.ops.layer_glue import residual_rms_norm
    from palimpsa_amd.ops.selective_scan import selective_scan
    from palimpsa_amd.ops.short_conv import short_conv
    gen = torch.Generator().manual_seed(T)
    D, N, W, S = 48, 16, 4, B if cu is None else len(cu) - 1
    inp = block_inputs(gen, B, T, D, N, W, S)
    cut = None if cu is None else torch.tensor(cu, device=gpu_device)
    own = (lambda x, r, w: residual_rms_norm(x, r, w, 1e-5),
           lambda x, w, b, s: short_conv(x, w, b, "silu", s, True, cut),
           lambda u, dl, A, B_, C, D_, z, b, h: selective_scan(u, dl, A, B_, C, D_, z, b, True, h, True, cut))
    plain = (lambda x, r, w: bo.residual_norm(x, r, w, 1e-5, torch.float64),
             lambda x, w, b, s: bo.conv(x, w, b, True, s, cu),
             lambda u, dl, A, B_, C, D_, z, b, h: bo.scan(u, dl, A, B_, C, D_, z, b, True, h, cu)[:2])
    cot = [torch.randn(B, T, D, generator=gen), torch.randn(S, D, W, generator=gen), torch.randn(S, D, N, generator=gen)]
    both = []
    for ops, to in ((own, lambda t: t.to(gpu_device)), (plain, lambda t: t.double())):
        lv = {n: to(t).requires_grad_(True) for n, t in inp.items()}
        out = block(lv, D, N, cu, ops)
        both.append([t.detach().cpu().double() for t in out + torch.autograd.grad(out, list(lv.values()), [to(t) for t in cot])])
    for i, (a, b) in enumerate(zip(*both)):
        assert (a - b).abs().max() <= 1e-3 * max(1.0, b.abs().max().item()), i


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_prompt_then_single_tokens_in_a_graph(gpu_device, dt):
    """Single tokens after a prompt, recorded once and replayed, against the whole sequence at once.  Both sides round the same values to
    the rows' type, and states are kept to what the kernels keep: in bf16 they may differ where fp32 sums of other orders fall on two sides
    of a rounding, one step (2^-8) of the largest value and as much again for what follows from it through conv, scan and gate (x 8)."""
    from palimpsa_amd.ops.layer_glue import residual_rms_norm
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step
    gen = torch.Generator().manual_seed(9)
    B, T, P, D, N, W = 3, 60, 41, 64, 16, 4
    a = {n: t.to(gpu_device) for n, t in block_inputs(gen, B, T, D, N, W, B).items()}
    a["x"], a["residual"] = a["x"].to(dt), a["residual"].to(dt)
    wp = a["wp"].to(dt)
    conv_state, scan_state = torch.zeros(B, D, W, dtype=dt, device=gpu_device), torch.zeros(B, D, N, device=gpu_device)

    def whole(x, res):
        y, res = residual_rms_norm(x, res, a["wn"], 1e-5)
        xs, z, dl, Bm, Cm = (y @ wp).split([D, D, D, N, N], -1)
        c, cf = short_conv(xs, a["wc"], a["bc"], output_final_state=True)
        o, hf = selective_scan(c, dl, a["A"], Bm, Cm, a["Dp"], z, a["bias"], output_final_state=True)
        return o + res, cf, hf

    def token(x, res):
        y, res = residual_rms_norm(x, res, a["wn"], 1e-5)
        xs, z, dl, Bm, Cm = (y @ wp).split([D, D, D, N, N], -1)
        c = short_conv_step(xs, conv_state, a["wc"], a["bc"])
        return selective_scan_step(c, scan_state, dl, a["A"], Bm, Cm, a["Dp"], z, a["bias"]) + res

    with torch.no_grad():
        want, _, hf = whole(a["x"], a["residual"])
        _, c0, h0 = whole(a["x"][:, :P], a["residual"][:, :P])
        xt, rt = torch.empty(B, D, dtype=dt, device=gpu_device), torch.empty(B, D, dtype=dt, device=gpu_device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            xt.copy_(a["x"][:, 0]), rt.copy_(a["residual"][:, 0])
            token(xt, rt)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = token(xt, rt)
        conv_state.copy_(c0), scan_state.copy_(h0)
        tol = 1e-3 if dt == torch.float32 else 2 * 8 * 2.0 ** -8
        for t in range(P, T):
            xt.copy_(a["x"][:, t]), rt.copy_(a["residual"][:, t])
            graph.replay()
            assert (out.float() - want[:, t].float()).abs().max() <= tol * max(1.0, want.float().abs().max().item()), t
        assert (scan_state - hf).abs().max() <= tol * max(1.0, hf.abs().max().item())


def test_convolutions_in_front_of_the_recurrence(gpu_device):
    """q, k and v go through a short convolution each and then into the framework's recurrence, with gradients back to the rows."""
    from palimpsa_amd.ops.palimpsa import chunk_palimpsa
    from palimpsa_amd.ops.short_conv import short_conv
    B, T, H, dk, dv, W = 2, 50, 2, 16, 16, 4
    inp = po.make_inputs(B, T, H, dk, dv, seed=4)
    gen = torch.Generator().manual_seed(1)
    filt = {n: torch.randn(H * d, W, generator=gen) / W for n, d in (("q", dk), ("k", dk), ("v", dv))}
    names = ("q", "k", "v", "b", "gt", "g", "Ip")

    def fwd(x, w, own):
        y = dict(x)
        for n in filt:
            c = (short_conv(x[n].flatten(2), w[n]) if own else bo.conv(x[n].flatten(2), w[n]))[0]
            y[n] = c.unflatten(2, (H, -1))
        return y

    lv = {n: inp[n].float().to(gpu_device).requires_grad_(True) for n in names}
    w = {n: t.to(gpu_device).requires_grad_(True) for n, t in filt.items()}
    y = fwd(lv, w, True)
    o = chunk_palimpsa(*[y[n] for n in names])
    cot = torch.randn(o.shape, generator=gen)
    got = torch.autograd.grad(o, [lv["q"], lv["k"], lv["v"], *w.values()], cot.to(gpu_device))
    # the plain form: the recurrence's gradients at the convolved rows, then through the plain convolution
    rows = {n: inp[n].double().requires_grad_(True) for n in names}
    wd = {n: t.double().requires_grad_(True) for n, t in filt.items()}
    yd = fwd(rows, wd, False)
    mid = {n: yd[n].detach().float().to(gpu_device).requires_grad_(True) for n in names}
    om = chunk_palimpsa(*[mid[n] for n in names])
    gm = torch.autograd.grad(om, [mid[n] for n in filt], cot.to(gpu_device))
    want = torch.autograd.grad([yd[n] for n in filt], [rows["q"], rows["k"], rows["v"], *wd.values()], [g.cpu().double() for g in gm])
    assert (o - om).abs().max() <= 1e-3 * max(1.0, om.abs().max().item())
    for a, b in zip(got, want):
        assert (a.cpu().double() - b).abs().max() <= 1e-3 * max(1.0, b.abs().max().item())
