"""Plain forms of the operators of a block's feed-forward half in 64 bits: dropout by counter, layer norm, gated feed-forward block, with the
formulas of their gradients.  Test infrastructure only."""
from __future__ import annotations

import math

import numpy as np
import torch


def philox(counter, key, rounds=7):
    """Philox4x32 (Salmon et al. 2011) of counters [.., 4] under a key of two words, in whole 64-bit products."""
    c = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    low, word = np.uint64(0xFFFFFFFF), np.uint64(32)
    key = list(key)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> word) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> word) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, -1)


def kept(shape, p, seed, site=0):
    """Truth values: which entries of [.., D] a dropout keeps."""
    D = shape[-1] if shape else 1
    rows = int(np.prod(shape[:-1], dtype=np.int64)) if shape else 1
    r, q = np.meshgrid(np.arange(rows, dtype=np.uint64), np.arange(-(-D // 4), dtype=np.uint64), indexing="ij")
    counter = np.stack([q, r & np.uint64(0xFFFFFFFF), r >> np.uint64(32), np.full_like(q, site)], -1)
    seed %= 2 ** 64
    words = philox(counter, (seed & 0xFFFFFFFF, seed >> 32)).reshape(rows, -1)[:, :D]
    least = min(math.floor(p * 2 ** 32 + 0.5), 2 ** 32 - 1)
    return torch.from_numpy(words >= np.uint64(least)).reshape(shape)


def layer_norm(s, weight, bias=None, eps=1e-5):
    """(y, normalised rows, 1 / sigma)."""
    s = s.double()
    mean = s.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    hat = (s - mean) * r
    y = hat * weight.double()
    return (y if bias is None else y + bias.double()), hat, r


def layer_norm_grads(dy, hat, r, weight):
    """(ds, dweight, dbias)."""
    dy = dy.double()
    gw = dy * weight.double()
    ds = r * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
    D = hat.shape[-1]
    return ds, (dy * hat).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)


def activation(name, g):
    """act(g), act'(g)."""
    if name == "silu":
        f = torch.sigmoid(g)
        return g * f, f * (1 + g * (1 - f))
    if name == "gelu":
        f = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * f, f + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    if name == "relu":
        return torch.where(g < 0, 0.0, g), (g > 0).to(g.dtype)
    raise ValueError(name)


def gated_mlp(x, w_gate, w_up, w_down, act="silu"):
    """(y, g, u, h) of rows [M, D]."""
    g, u = x @ w_gate.T, x @ w_up.T
    h = activation(act, g)[0] * u
    return h @ w_down.T, g, u, h


def gated_mlp_grads(dy, x, w_gate, w_up, w_down, act="silu"):
    """(dx, dw_gate, dw_up, dw_down)."""
    _, g, u, h = gated_mlp(x, w_gate, w_up, w_down, act)
    a, d = activation(act, g)
    dh = dy @ w_down
    dg, du = dh * u * d, dh * a
    return dg @ w_gate + du @ w_up, dg.T @ x, du.T @ x, dy.T @ h
