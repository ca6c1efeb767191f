"""Sizes that between them take every tile form of the gated feed-forward block's products, in every round and share that the plan gives it, and data on which
the results are exact."""
from __future__ import annotations

import torch

PRODUCTS = ("up", "down", "grad", "dx", "dw")
STEP = {"bf16": 64, "fp32": 32}          # k of a step
SIZES = {                                # rows, dim, hidden, out_dim
    "bf16": [(935, 542, 197, 164), (168, 249, 2056, 748), (39591, 526, 144, 173), (22126, 1670, 8, 1101), (53986, 130, 197, 271), (30801, 1185, 174, 400),
             (16638, 11, 1993, 151), (32877, 251, 338, 299), (10480, 161, 5422, 398), (10953, 8, 133, 2282), (159, 2850, 5530, 1860), (1700, 2385, 1677, 16),
             (36313, 135, 1861, 21), (131, 2572, 2129, 128), (39373, 276, 68, 32), (133, 1299, 4909, 149), (131, 1540, 4957, 16), (11079, 507, 5063, 30)],
    "fp32": [(78, 82, 65, 75), (74, 624, 1803, 463), (27381, 77, 76, 82), (4150, 90, 1508, 65), (4230, 1327, 94, 2891), (18367, 65, 2015, 94),
             (16709, 1341, 81, 1146), (12360, 172, 1271, 215), (59091, 143, 100, 152), (351, 1878, 2907, 108), (8501, 1782, 85, 2803), (2197, 2092, 4682, 1236),
             (1010, 1787, 5695, 2431), (20641, 730, 240, 1527), (32551, 980, 71, 492), (25727, 544, 65, 1703), (1787, 2520, 2175, 1791), (8692, 169, 3721, 508),
             (16909, 17, 4107, 129), (65, 1349, 4019, 122), (73, 2710, 5556, 16), (24073, 442, 715, 2696), (2247, 36, 2756, 2851)],
}
# those of the training batch, the prompt and the fp32 step that the notes have times of, and of few rows
KNOWN = {"bf16": [(16384, 768, 2048, 768), (8192, 2048, 5632, 2048), (48, 2048, 5632, 2048)], "fp32": [(1503, 771, 2058, 771), (4096, 1024, 2816, 1024)]}
FEW = [(1, 768, 2048, 768), (3, 61, 97, 39), (16, 2048, 1408, 520), (17, 136, 704, 136), (32, 512, 1408, 512), (33, 768, 2048, 768), (48, 61, 97, 39), (64, 256, 704, 256)]


def forms(L, M, D, F, Do, dtype):
    """{product: (rows of a tile, columns, shares of k, tiles)} of a forward and backward; nothing of a product by the kernels of few rows."""
    import ctypes as C
    up8 = lambda n: -(-n // 8) * 8  # noqa: E731
    P, f = C.c_void_p(0x1000), L.PalMlpForms()
    d = L.PalMlpDims(rows=M, x_stride=up8(D), dim=up8(D), hidden=up8(F), out_dim=up8(Do), dtype=int(dtype == "bf16"), activation=3, hidden_pad=up8(F) - F)
    assert L.load().pal_gated_mlp_forms(d, L.PalMlpGrads(dy=P, dx=P, dw_gate=P, dw_up=P, dw_down=P), f) == 0
    return {n: (f.tile_rows[i], f.tile_cols[i], f.shares[i], f.tiles[i]) for i, n in enumerate(PRODUCTS) if f.tile_rows[i]}


def taken(L, M, D, F, Do, dtype):
    """{(product, rows of a tile, columns, k in shares, workgroups with more than one tile)} with three steps of k or more, the last of them cut short."""
    out, per = set(), STEP[dtype]
    for n, (m, c, shares, tiles) in forms(L, M, D, F, Do, dtype).items():
        k = {"up": D, "down": F, "grad": Do, "dx": F, "dw": M}[n]
        steps = -(-k // per) * (2 if n == "dx" else 1) // shares
        if steps >= 3 and k % per:
            out.add((n, m, c, shares > 1, tiles * shares > {256: 256, 128: 512, 64: 1024}[m]))
    return out


def whole_numbers(dev, M, D, F, Do, dtype, seed=0):
    """x, w_gate, w_up, w_down, dy of -1, 0 and 1, thin enough that every sum on the way is a whole number that fp32 and the kept factors hold exactly."""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def thin(rows, cols, share):
        r = torch.rand(rows, cols, generator=gen, device=dev)
        return ((r < share / 2).to(dtype) - (r >= 1 - share / 2).to(dtype))

    w = min(1.0, 64 / D)
    return thin(M, D, 0.25), thin(F, D, w), thin(F, D, w), thin(Do, F, min(1.0, 64 / max(F, Do))), thin(M, Do, 0.25)


def exact(x, wg, wu, wd, dy, dtype):
    """y and the four gradients with relu as the kernels have to give them: products exact, h, dg and du rounded to the type of the rows (h of up to 16 rows is a
    sum of two numbers), results rounded once."""
    few, wide = x.shape[0] <= 16, [t.double() for t in (x, wg, wu, wd, dy)]
    x, wg, wu, wd, dy = wide
    stored = lambda t: t.to(dtype).double()  # noqa: E731
    least = 2.0 ** 24
    g, u = x @ wg.T, x @ wu.T
    a = g.clamp(min=0)
    h = a * u
    dh = dy @ wd
    dg, du = stored(dh * u * (g > 0)), stored(dh * a)
    hr = stored(h)
    for t in (g, u):
        assert t.abs().max() < 1024                                     # kept exactly, and h a sum of two bf16 numbers
    assert h.abs().max() < 2 ** 16 and (dh * u).abs().max() < least
    out = []
    for terms in (([h if few else hr], [wd.T]), ([dg, du], [wg, wu]), ([dg.T], [x]), ([du.T], [x]), ([dy.T], [hr])):
        pairs = list(zip(*terms))
        assert sum(p.abs() @ q.abs() for p, q in pairs).max() < least   # any order of the sums is exact
        out.append(sum(p @ q for p, q in pairs).to(dtype))
    return out
