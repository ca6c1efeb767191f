"""Plain 64-bit forms of the operators around the recurrences: short causal convolution, selective scan, residual norm.

Test infrastructure only.  Every function computes in float64 on the CPU (or wherever its inputs are), token by token where
the operator is a recurrence, and takes packed batches as a list of sequence bounds.  The backward passes are written out from
the formulas; the tests hold them against automatic differentiation and differences.  With ``mass`` every product is taken of absolute
values: the sum of the sizes of all terms behind a result, which is what its rounding error is a multiple of.
"""
from __future__ import annotations

import torch


def bounds(B, T, cu=None):
    """(batch row, first token, end) of every sequence."""
    return [(b, 0, T) for b in range(B)] if cu is None else [(0, cu[i], cu[i + 1]) for i in range(len(cu) - 1)]


# ------------------------------------------------------------------------------------------------- short convolution
def conv(x, weight, bias=None, silu=True, init=None, cu=None):
    """(y, final states [N, D, W]); differentiable."""
    x, weight = x.double(), weight.double()
    B, T, D = x.shape
    W = weight.shape[1]
    y, finals = torch.zeros_like(x), []
    for n, (b, s, e) in enumerate(bounds(B, T, cu)):
        old = x.new_zeros(W, D) if init is None else init[n].double().T
        line = torch.cat([old, x[b, s:e]])
        p = sum(weight[:, k] * line[1 + k:1 + k + e - s] for k in range(W))
        if bias is not None:
            p = p + bias.double()
        y = torch.index_put(y, (torch.tensor([b]).view(1, 1), torch.arange(s, e).view(1, -1)),
                            (p * torch.sigmoid(p) if silu else p).unsqueeze(0)) if e > s else y
        finals.append(line[e - s:].T)
    return y, torch.stack(finals)


# ----------------------------------------------------------------------------------------------------- selective scan
def step_size(delta, delta_bias, softplus):
    raw = delta.double() + (0 if delta_bias is None else delta_bias.double())
    return torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20)))) if softplus else raw


def _wide(t, ch):
    """[B, T, N] or [B, T, G, N] -> [B, T, channels, N]"""
    t = t.double()
    t = t.unsqueeze(2) if t.dim() == 3 else t
    return t.repeat_interleave(ch // t.shape[2], 2)


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, init=None, cu=None, mass=False):
    """(y, final states, states after every token, sum_n C h + D u); differentiable without ``mass``."""
    f = torch.abs if mass else (lambda t: t)
    ch, N = A.shape
    bt, T = u.shape[:2]
    dt = step_size(delta, delta_bias, softplus)
    Bw, Cw = f(_wide(B, ch)), f(_wide(C, ch))
    x = f(dt * u.double())
    states, finals, rows = [[None] * T for _ in range(bt)], [], []
    for n, (b, s, e) in enumerate(bounds(bt, T, cu)):
        h = torch.zeros(ch, N, dtype=torch.float64, device=u.device) if init is None else f(init[n].double())
        for t in range(s, e):
            h = torch.exp(dt[b, t, :, None] * A.double()) * h + x[b, t, :, None] * Bw[b, t]
            states[b][t] = h
        finals.append(h)
    H = torch.stack([torch.stack(r) for r in states])
    pre = (H * Cw).sum(-1)
    if D is not None:
        pre = pre + f(D.double() * u.double())
    y = pre if z is None else pre * f(z.double() * torch.sigmoid(z.double()))
    return y, torch.stack(finals), H, pre


def scan_grads(dy, u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, init=None, cu=None, d_final=None, mass=False):
    """Gradients of sum(y * dy) + sum(final * d_final) by the formulas: a dict of du, ddelta, dA, dB, dC, dD, dz, ddelta_bias, d_init."""
    f = torch.abs if mass else (lambda t: t)
    ch, N = A.shape
    bt, T = u.shape[:2]
    _, _, H, pre = scan(u, delta, A, B, C, D, z, delta_bias, softplus, init, cu, mass)
    raw = delta.double() + (0 if delta_bias is None else delta_bias.double())
    dt = step_size(delta, delta_bias, softplus)
    Bw, Cw, Af, ud, dy = f(_wide(B, ch)), f(_wide(C, ch)), f(A.double()), f(u.double()), f(dy.double())
    G = B.shape[2] if B.dim() == 4 else 1
    out = {}
    Y = dy
    if z is not None:
        zd, sg = z.double(), torch.sigmoid(z.double())
        Y = dy * f(zd * sg)
        # silu' is a sum of two terms, of opposite sign for z < 0: near its zero at -1.28 it is s - s, each rounded by itself, so that
        # the size of its terms is their sum (0.44 there) and not the difference
        out["dz"] = dy * pre * (sg + f(zd) * sg * (1 - sg))
    x = f(dt * u.double())
    du, ddt, dA = torch.zeros_like(dt), torch.zeros_like(dt), torch.zeros(ch, N, dtype=torch.float64, device=u.device)
    dBw, dCw, d_init = torch.zeros_like(H), torch.zeros_like(H), []
    for n, (b, s, e) in enumerate(bounds(bt, T, cu)):
        g = torch.zeros(ch, N, dtype=torch.float64, device=u.device) if d_final is None else f(d_final[n].double())
        for t in range(e - 1, s - 1, -1):
            a = torch.exp(dt[b, t, :, None] * A.double())
            g = g + Cw[b, t] * Y[b, t, :, None]
            before = H[b, t - 1] if t > s else torch.zeros_like(g) if init is None else f(init[n].double())
            ah = a * before
            dCw[b, t] = Y[b, t, :, None] * H[b, t]
            dBw[b, t] = g * x[b, t, :, None]
            sB = (g * Bw[b, t]).sum(-1)
            du[b, t] = f(dt[b, t]) * sB
            ddt[b, t] = (g * ah * Af).sum(-1) + ud[b, t] * sB
            dA += g * ah * f(dt[b, t])[:, None]
            g = a * g
        d_init.append(g)
    if D is not None:
        du = du + f(D.double()) * Y
        out["dD"] = (Y * ud).sum((0, 1))
    dd = ddt * torch.sigmoid(raw) if softplus else ddt
    if softplus:
        dd = torch.where(raw > 20, ddt, dd)
    sums = lambda v: v.reshape(bt, T, G, ch // G, N).sum(3).reshape(B.shape)  # noqa: E731
    out.update(du=du, ddelta=dd, dA=dA, dB=sums(dBw), dC=sums(dCw), d_init=torch.stack(d_init))
    if delta_bias is not None:
        out["ddelta_bias"] = dd.sum((0, 1))
    return out


# ----------------------------------------------------------------------------------------------------- residual norm
def residual_norm(x, residual, weight, eps, res_dtype):
    """(y, stream as it is handed on); the stream is rounded to its type, straight through for gradients."""
    s = x.double() if residual is None else x.double() + residual.double()
    s = s + (s.detach().float().to(res_dtype).double() - s.detach())
    r = torch.rsqrt((s * s).mean(-1, keepdim=True) + eps)
    return s * r * weight.double(), s
