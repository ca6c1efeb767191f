"""Bounds of the errors of the feed-forward half's operators, from the roundings that their kernels make: half a step of the rows' type for
each tensor that is stored in it, 2^-24 per operation for what is done in fp32."""
from __future__ import annotations

import torch

from oracle import feed_forward_oracle as fo

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gated_mlp(x, wg, wu, wd, act, dtype, dy=None):
    """({name: value}, {name: bound}) in 64 bits on the inputs as given; y, and with dy the gradients."""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    ax, ag, au, ad = (t.abs() for t in (x, wg, wu, wd))
    y, g, u, h = fo.gated_mlp(x, wg, wu, wd, act)
    a, d = fo.activation(act, g)
    r, (M, D), F, Do = half_step(dtype), x.shape, wg.shape[0], wd.shape[0]
    # sums in fp32: at most one rounding per term; the activation by a reciprocal and an exponential of one or two units each, whose
    # argument's rounding counts with its size, and erf's of a few units: (|g| + 8) 2^-23 of the factor that multiplies g
    eg, eu = D * E32 * (ax @ ag.T), D * E32 * (ax @ au.T)
    slope = 1.13                                                   # the steepest of the activations
    ea = slope * eg + g.abs() * (g.abs() + 8) * 2 * E32
    eh = ea * u.abs() + a.abs() * eu + h.abs() * (r + 2 * E32)
    # up to 16 rows h is the sum of two numbers of the type: half a step of what half a step leaves
    ey = ea * u.abs() + a.abs() * eu + h.abs() * (r * r + 2 * E32) if M <= 16 and dtype == torch.bfloat16 else eh
    terms = F if ey is eh else 2 * F
    val = {"y": y}
    tol = {"y": ey @ ad.T + terms * E32 * (h.abs() @ ad.T) + r * y.abs()}
    if dy is None:
        return val, tol
    dy = dy.detach().double()
    dh = dy @ wd
    edh = Do * E32 * (dy.abs() @ ad)
    # g and u are kept with nine bits after the leading one, rounded to the nearest: half a step is at most 2^-10 of the number; where that is
    # below fp16's 2^-14, the largest of its eight being 2^14 or more, half a step is 2^-24, 2^-38 of the largest
    if dtype == torch.bfloat16:
        def step(t):
            n = -t.shape[1] % 8
            top = torch.nn.functional.pad(t.abs(), (0, n)).reshape(M, -1, 8).amax(2, keepdim=True)
            return 2.0 ** -10 * t.abs() + 2.0 ** -38 * top.expand(-1, -1, 8).reshape(M, -1)[:, :t.shape[1]]
        eg, eu = eg + step(g), eu + step(u)
    ea = slope * eg + g.abs() * (g.abs() + 8) * 2 * E32
    bend = 0.8                                                     # the largest second derivative
    ed = bend * eg + (1 + g.abs()) * (g.abs() + 8) * 4 * E32
    if act == "relu":
        ed = ed + (g.abs() <= eg).double()                         # its derivative jumps at 0
    dg, du = dh * u * d, dh * a
    edg = edh * (u * d).abs() + dh.abs() * (eu * d.abs() + u.abs() * ed) + dg.abs() * (r + 4 * E32)
    edu = edh * a.abs() + dh.abs() * ea + du.abs() * (r + 2 * E32)
    val.update(x=dg @ wg + du @ wu, w_gate=dg.T @ x, w_up=du.T @ x, w_down=dy.T @ h)
    tol["x"] = edg @ ag + edu @ au + 2 * F * E32 * (dg.abs() @ ag + du.abs() @ au) + r * val["x"].abs()
    tol["w_gate"] = edg.T @ ax + M * E32 * (dg.abs().T @ ax) + r * val["w_gate"].abs()
    tol["w_up"] = edu.T @ ax + M * E32 * (du.abs().T @ ax) + r * val["w_up"].abs()
    tol["w_down"] = dy.abs().T @ eh + M * E32 * (dy.abs().T @ h.abs()) + r * val["w_down"].abs()
    return val, tol


def layer_norm(s, w, b, eps, dtype, dy=None, dres=None):
    """The same of a layer norm of s as it was handed on: y, and with dy ds (before any dropout), dweight, dbias."""
    y, hat, r = fo.layer_norm(s, w, b, eps)
    s, w = s.double(), w.double()
    n = 80 * E32               # a lane's sum of at most 64 entries and the tree over lanes and waves
    size = s.abs() + s.abs().mean(-1, keepdim=True)
    # the mean's error moves the rows, that of the variance scales them
    ehat = r * n * size + hat.abs() * (n + 2 * (n * r * size).mean(-1, keepdim=True) + 8 * E32)
    val = {"y": y}
    tol = {"y": half_step(dtype) * y.abs() + ehat * w.abs() + 2 * E32 * (0 if b is None else b.double().abs()) + 4 * E32 * y.abs()}
    if dy is None:
        return val, tol
    ds, dw, db = fo.layer_norm_grads(dy, hat, r, w)
    dy = dy.double()
    gw = (dy * w).abs()
    er = r * (n + 2 * (n * r * size).mean(-1, keepdim=True) + 8 * E32)        # of 1 / sigma
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    inner = gw + mean(gw) + hat.abs() * mean(gw * hat.abs())
    eds = er * inner + r * (n * inner + ehat * mean(gw * hat.abs()) + hat.abs() * mean(gw * ehat))
    if dres is not None:
        ds = ds + dres.double()
    eds = eds + 2 * E32 * ds.abs()
    D, rows = s.shape[-1], s.numel() // s.shape[-1]
    flat = lambda t: t.reshape(-1, D).sum(0)  # noqa: E731
    val.update(ds=ds, weight=dw, bias=db)
    tol.update(ds=eds, weight=(rows + 8) * E32 * flat((dy * hat).abs()) + flat(dy.abs() * ehat), bias=(rows + 8) * E32 * flat(dy.abs()))
    return val, tol


def within(got, want, tol, what):
    err = (got.detach().double() - want).abs()
    bad = ~(err <= tol)
    if bad.any():
        i = int((err - tol).nan_to_num(float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} entries off, e.g. [{i}] {got.reshape(-1)[i].item()} instead of "
                             f"{want.reshape(-1)[i].item()}, allowed {tol.reshape(-1)[i].item():.3g}")
