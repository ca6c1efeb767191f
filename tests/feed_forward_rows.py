"""Places of a dropout from explicit row numbers, on any device, and bounds of the sums over many rows."""
from __future__ import annotations

import math

import torch

E32 = 2.0 ** -24


def kept(row, D, p, seed, site=0):
    """Truth values [rows, D] of the rows with these numbers (int64): Philox4x32 with seven rounds, products of 32 bits from halves of one factor."""
    def mul(m, a):
        top, low = (a >> 16) * m, (a & 0xFFFF) * m
        mid = top + (low >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    quads, seed = -(-D // 4), seed % 2 ** 64
    c0 = torch.arange(quads, device=row.device).expand(row.numel(), quads)
    c1, c2 = ((row & 0xFFFFFFFF)[:, None].expand_as(c0), (row >> 32)[:, None].expand_as(c0))
    c3 = torch.full_like(c0, site)
    for i in range(7):
        k0, k1 = ((seed & 0xFFFFFFFF) + i * 0x9E3779B9) % 2 ** 32, ((seed >> 32) + i * 0xBB67AE85) % 2 ** 32
        (h0, l0), (h1, l1) = mul(0xD2511F53, c0), mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
    words = torch.stack([c0, c1, c2, c3], 2).reshape(row.numel(), 4 * quads)[:, :D]
    return words >= min(math.floor(p * 2 ** 32 + 0.5), 2 ** 32 - 1)


def dropped(t, p, seed, site=0, first=0):
    """Kept entries of the rows from number `first` on times the scale in fp32, in 64 bits."""
    if not p:
        return t.double()
    rows = t.reshape(-1, t.shape[-1])
    keep = kept(torch.arange(first, first + rows.shape[0], device=t.device), t.shape[-1], p, seed, site).reshape(t.shape)
    return torch.where(keep, t.double() * (1 / (1 - p)), 0.0)


def depth(rows, D):
    """Additions that a term of dweight or dbias passes through: a wave's rows one by one (at least 256 workgroups of four waves with a row each, or of one
    row), four waves, then the workgroups' shares (up to 1024) by 64 groups, and two rounds of eight of these."""
    return -(-rows // (256 * (4 if D <= 2048 else 1))) + 4 + 16 + 16 + 1
