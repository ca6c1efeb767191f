"""The operators of the feed-forward half of a block, as cases to be timed: the layer norm (alone, or with the residual's addition and
a dropout in front of it), dropout by itself, and the gated feed-forward block, in training, for prompts and for a few tokens.

Shapes are those of the layer configurations that the repository's tests and notes name (rows of 768 and 1536, batches of 8 x 2048) with the
hidden sizes that such layers take (two thirds of four times the row, in multiples of 256), and generic ones of the same kind in
`draw`.  A case is one pass of one `op` in one `form`:

* mlp   ``train`` forward + backward, ``serve`` forward;  y = (act(x Wg^T) * (x Wu^T)) Wd^T
* norm  the same two; with ``res`` the rows are added to a residual stream first (after a dropout of probability ``p``), which is handed on
* drop  the same two; entries are kept by a counter-based generator, from the seed, the row and the column alone

`own` is set by whoever runs the cases: False computes each operator from elementary torch operations, True calls the framework.
"""
import math

import numpy as np
import torch

own = False

# no drawn case multiplies, normalises or drops more than the largest listed one of its operator
MOST = {"mlp": 8192 * 2048 * 5632, "norm": 16384 * 1536, "drop": 16384 * 2048}
ACTS = ("silu", "gelu", "gelu_tanh", "relu")
EPS = 1e-5


def _case(name, op, form, B, T, D, dtype="bf16", F=0, act="silu", res=None, bias=True, p=0.0):
    """``F``: hidden size of the feed-forward block; ``res``: type of the residual stream (None: a norm without one); ``bias``: the norm
    adds one; ``p``: probability of being dropped."""
    c = dict(op=op, form=form, B=B, T=T, D=D, dtype=dtype, F=F, act=act, res=res, bias=bias, p=p)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one conversation, token by token: all latency
        _case("mlp_step", "mlp", "serve", 1, 1, 768, F=2048),
        # a serving batch of 48 conversations, one token each: the weights are all the traffic
        _case("mlp_decode", "mlp", "serve", 48, 1, 2048, F=5632),
        # a long prompt read in
        _case("mlp_prompt", "mlp", "serve", 1, 8192, 2048, F=5632),
        # training batch of a small model
        _case("mlp_train", "mlp", "train", 8, 2048, 768, F=2048),
        # odd sizes in full precision, another activation: a check of a layer
        _case("mlp_fp32", "mlp", "train", 3, 501, 771, dtype="fp32", F=2058, act="gelu"),
        # a small decode batch through the norm between two blocks
        _case("norm_serve", "norm", "serve", 16, 1, 768, res="bf16"),
        # training batch: dropout, addition to an fp32 stream and norm of it
        _case("norm_train", "norm", "train", 8, 2048, 1536, res="fp32", p=0.1),
        # a norm by itself, odd row length, fp32
        _case("norm_fp32", "norm", "train", 1, 4099, 1531, dtype="fp32"),
        # dropout of a training batch's rows
        _case("drop_train", "drop", "train", 8, 2048, 2048, p=0.1),
        # the same of odd rows in fp32
        _case("drop_fp32", "drop", "train", 3, 1001, 771, dtype="fp32", p=0.25),
        # a few rows, sampled at inference (an ensemble by dropout)
        _case("drop_serve", "drop", "serve", 16, 1, 768, p=0.1),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["mlp", "norm", "drop"])
        form = rng.choice(["train", "serve"])
        dtype = "fp32" if rng.random() < 0.3 else "bf16"
        B, T = _between(rng, 1, 16), _between(rng, 1, 8192)
        if form == "serve" and rng.random() < 0.4:
            B, T = _between(rng, 1, 256), 1
        D = rng.choice([_between(rng, 16, 2048), 8 * _between(rng, 4, 256)])
        F, act, res, bias, p = 0, "silu", None, True, 0.0
        size = B * T * D
        if op == "mlp":
            F = rng.choice([_between(rng, 32, 5632), 8 * _between(rng, 8, 704)])
            act = rng.choice(ACTS)
            size *= F * (10 if dtype == "fp32" else 1) * (3 if form == "train" else 1)
        elif op == "norm":
            res = rng.choice([None, "fp32", "fp32" if dtype == "fp32" else "bf16"])
            bias = rng.random() < 0.7
            p = rng.choice([0.0, 0.1, 0.5]) if res else 0.0
            size *= 2 if dtype == "fp32" else 1
        else:
            p = rng.choice([0.05, 0.1, 0.25, 0.5])
            size *= 2 if dtype == "fp32" else 1
        if size <= MOST[op]:
            return _case(None, op, form, B, T, D, dtype, F, act, res, bias, p)


def _dtype(name):
    return torch.float32 if name == "fp32" else torch.bfloat16


def prepare(c, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    B, T, D, F, dt = c["B"], c["T"], c["D"], c["F"], _dtype(c["dtype"])
    normal = lambda *shape, dtype=dt: torch.randn(*shape, generator=gen, device=dev).to(dtype)  # noqa: E731
    uniform = lambda lo, hi, *shape: lo + (hi - lo) * torch.rand(*shape, generator=gen, device=dev)  # noqa: E731
    s = {"op": c["op"], "form": c["form"], "act": c["act"], "p": c["p"], "leaves": {}}
    # what a program draws for a step, and the number of the place in the model
    s["seed"], s["site"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63), seed % 7
    x = s["leaves"]
    x["x"] = normal(B, T, D)                 # rows as a norm in front of the block gives them
    if c["op"] == "mlp":
        # weights as a linear layer's are initialised
        x.update(w_gate=(uniform(-1, 1, F, D) / math.sqrt(D)).to(dt), w_up=(uniform(-1, 1, F, D) / math.sqrt(D)).to(dt),
                 w_down=(uniform(-1, 1, D, F) / math.sqrt(F)).to(dt))
    elif c["op"] == "norm":
        if c["res"]:
            x["residual"] = (3.0 * normal(B, T, D, dtype=torch.float32) + 0.5).to(_dtype(c["res"]))
        x["weight"] = uniform(0.5, 1.5, D)
        if c["bias"]:
            x["bias"] = uniform(-0.5, 0.5, D)
    if c["form"] == "train":
        s["dy"] = normal(B, T, D)
        if c["res"]:
            s["dres"] = normal(B, T, D, dtype=_dtype(c["res"]))
        for t in x.values():
            t.requires_grad_(True)
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"mlp": _mlp, "norm": _norm, "drop": _drop}[s["op"]](s)


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    if s["form"] == "train":
        out = _own_forward(s)
        grads = torch.autograd.grad(out, list(s["leaves"].values()), [s["dy"], s["dres"]] if "dres" in s else [s["dy"]])
        return {"out": [o.detach() for o in out], "grads": list(grads)}
    with torch.no_grad():
        return {"out": _own_forward(s)}


def _own_forward(s):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm, residual_layer_norm

    x = s["leaves"]
    if s["op"] == "mlp":
        return [gated_mlp(**x, activation=s["act"])]
    if s["op"] == "drop":
        return [dropout(x["x"], s["p"], s["seed"], s["site"])]
    if "residual" not in x:
        return [layer_norm(**x, eps=EPS)]
    if s["p"]:
        return list(residual_layer_norm(**x, eps=EPS, dropout_p=s["p"], seed=s["seed"], site=s["site"]))
    return list(residual_layer_norm(**x, eps=EPS))


# ------------------------------------------------------------------------------------------------------- the plain forms
def _activation(act, g):
    """act(g) and its derivative."""
    if act == "silu":
        f = torch.sigmoid(g)
        return g * f, f * (1 + g * (1 - f))
    if act == "gelu":
        f = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * f, f + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), (g > 0).to(g.dtype)


def _mlp(s):
    x, dt = s["leaves"], s["leaves"]["x"].dtype
    rows, wg, wu, wd = (x[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    rows = rows.reshape(-1, rows.shape[-1])
    g, u = rows @ wg.T, rows @ wu.T
    a, da = _activation(s["act"], g)
    h = a * u
    y = (h @ wd.T).to(dt).reshape(x["x"].shape)
    if s["form"] == "serve":
        return {"out": [y]}
    dy = s["dy"].float().reshape(-1, wd.shape[0])
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    dx = dg @ wg + du @ wu
    grads = [dx.reshape(x["x"].shape), dg.T @ rows, du.T @ rows, dy.T @ h]
    return {"out": [y], "grads": [t.to(dt) for t in grads]}


def _philox(c0, c1, c2, c3, k0, k1, rounds=7):
    """Four words of 32 bits for a counter of four and a key of two (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011), in
    64-bit integers: the products of two words are put together from halves of one."""
    def mul(m, a):
        top, low = (a >> 16) * m, (a & 0xFFFF) * m
        mid = top + (low >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    for i in range(rounds):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ ((k0 + i * 0x9E3779B9) & 0xFFFFFFFF), l1, h0 ^ c3 ^ ((k1 + i * 0xBB67AE85) & 0xFFFFFFFF), l0
    return c0, c1, c2, c3


def _kept(s, rows, D, dev):
    """Truth values [rows, D]: the entry's word is not below p 2^32."""
    quads = (D + 3) // 4
    q = torch.arange(quads, device=dev).expand(rows, quads)
    r = torch.arange(rows, device=dev).unsqueeze(1).expand(rows, quads)
    w = _philox(q, r & 0xFFFFFFFF, r >> 32, torch.full_like(q, s["site"]), s["seed"] & 0xFFFFFFFF, s["seed"] >> 32)
    return torch.stack(w, 2).reshape(rows, 4 * quads)[:, :D] >= round(s["p"] * 2 ** 32)


def _drop(s):
    x = s["leaves"]["x"]
    D, scale = x.shape[-1], 1 / (1 - s["p"])
    keep = _kept(s, x.numel() // D, D, x.device).reshape(x.shape)
    dropped = lambda t: torch.where(keep, t.float() * scale, 0.0).to(t.dtype)  # noqa: E731
    if s["form"] == "serve":
        return {"out": [dropped(x)]}
    return {"out": [dropped(x)], "grads": [dropped(s["dy"])]}


def _norm(s):
    leaves = s["leaves"]
    x, res, w, b = (leaves.get(n) for n in ("x", "residual", "weight", "bias"))
    D = w.numel()
    rows, new = x.float(), x
    if s["p"]:
        keep = _kept(s, x.numel() // D, D, x.device).reshape(x.shape)
        rows = torch.where(keep, rows * (1 / (1 - s["p"])), 0.0)
    if res is not None:
        new = (rows + res.float()).to(res.dtype)
    v = new.float()
    v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    hat = v * r
    y = (hat * w if b is None else hat * w + b).to(x.dtype)
    out = [y] if res is None else [y, new]
    if s["form"] == "serve":
        return {"out": out}
    gy = s["dy"].float()
    gw = gy * w
    dv = r * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
    if res is not None:
        dv = dv + s["dres"].float()
    grads = [(torch.where(keep, dv * (1 / (1 - s["p"])), 0.0) if s["p"] else dv).to(x.dtype)]
    if res is not None:
        grads.append(dv.to(res.dtype))
    sums = [(gy * hat).reshape(-1, D).double().sum(0).float()]
    if b is not None:
        sums.append(gy.reshape(-1, D).double().sum(0).float())
    return {"out": out, "grads": grads + sums}


# ----------------------------------------------------------------------------------------------------------- 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"mlp": _exact_mlp, "norm": _exact_norm, "drop": _exact_drop}[c["op"]](s)


def _exact_mlp(s):
    x = s["leaves"]
    X, G, U, W = (x[n].double() for n in ("x", "w_gate", "w_up", "w_down"))
    D, act = X.shape[-1], s["act"]
    X = X.reshape(-1, D)
    g, u = torch.mm(X, G.t()), torch.mm(X, U.t())
    if act == "silu":
        a = g / (1 + torch.exp(-g))
        slope = (1 + torch.exp(-g) + g * torch.exp(-g)) / (1 + torch.exp(-g)) ** 2
    elif act == "gelu":
        below = 0.5 * torch.erfc(-g / 2 ** 0.5)
        a, slope = g * below, below + g * torch.exp(-g * g / 2) / (2 * math.pi) ** 0.5
    elif act == "gelu_tanh":
        z = (8 / math.pi) ** 0.5 * (g + 0.044715 * g * g * g)       # (1 + tanh(z / 2)) / 2 = 1 / (1 + e^-z)
        f = 1 / (1 + torch.exp(-z))
        a, slope = g * f, f + g * f * (1 - f) * (8 / math.pi) ** 0.5 * (1 + 0.134145 * g * g)
    else:
        a, slope = torch.where(g > 0, g, 0.0), torch.where(g > 0, 1.0, 0.0).double()
    y = torch.mm(a * u, W.t()).reshape(x["x"].shape)
    if s["form"] == "serve":
        return {"out": [y]}
    dy = s["dy"].double().reshape(-1, D)
    dh = torch.mm(dy, W)
    dW = torch.mm(dy.t(), a * u)
    dg, du = dh * u * slope, dh * a
    dx = torch.mm(dg, G) + torch.mm(du, U)
    return {"out": [y], "grads": [dx.reshape(x["x"].shape), torch.mm(dg.t(), X), torch.mm(du.t(), X), dW]}


def _exact_kept(s, shape, dev):
    """The same truth values from whole 64-bit products, on the host."""
    D, word, low = shape[-1], np.uint64(32), np.uint64(0xFFFFFFFF)
    rows = int(np.prod(shape[:-1]))
    r, q = np.meshgrid(np.arange(rows, dtype=np.uint64), np.arange(-(-D // 4), dtype=np.uint64), indexing="ij")
    c = [q, r & low, r >> word, np.full_like(q, s["site"])]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> word) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> word) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(c, -1).reshape(rows, -1)[:, :D]
    return torch.from_numpy(words >= np.uint64(round(s["p"] * 2 ** 32))).to(dev).reshape(shape)


def _exact_drop(s):
    x = s["leaves"]["x"]
    factor = _exact_kept(s, x.shape, x.device).double() / (1 - s["p"])
    if s["form"] == "serve":
        return {"out": [x.double() * factor]}
    return {"out": [x.double() * factor], "grads": [s["dy"].double() * factor]}


def _exact_norm(s):
    leaves = s["leaves"]
    x, res, w, b = (leaves.get(n) for n in ("x", "residual", "weight", "bias"))
    factor = _exact_kept(s, x.shape, x.device).double() / (1 - s["p"]) if s["p"] else 1.0
    v = x.double() * factor
    out = []
    if res is not None:
        v = (v + res.double()).to(res.dtype).double()         # the stream is handed on in its own type
        out = [v]
    D = w.numel()
    w = w.double()
    mean = v.sum(-1, keepdim=True) / D
    sigma = torch.sqrt(((v - mean) ** 2).sum(-1, keepdim=True) / D + EPS)
    hat = (v - mean) / sigma
    y = hat * w + (0.0 if b is None else b.double())
    if s["form"] == "serve":
        return {"out": [y] + out}
    gy = s["dy"].double()
    gw = gy * w
    dv = (gw - gw.sum(-1, keepdim=True) / D - hat * (gw * hat).sum(-1, keepdim=True) / D) / sigma
    sums = [(gy * hat).reshape(-1, D).sum(0)] + ([] if b is None else [gy.reshape(-1, D).sum(0)])
    if res is None:
        return {"out": [y], "grads": [dv] + sums}
    dv = dv + s["dres"].double()
    return {"out": [y] + out, "grads": [dv * factor, dv] + sums}


def work(c):
    """Each tensor of the call read or written once, and the operations of the formulas: a feed-forward block three products of 2 per row,
    entry and hidden entry, its backward six; a norm 8 per entry, backward 14 more (with dropout 20 more each way: seven rounds of two
    wide products, two sums of keys and four exclusive ors for four entries, the comparison and the product); a dropout those 20."""
    B, T, D, F = c["B"], c["T"], c["D"], c["F"]
    e, r = (4 if c["dtype"] == "fp32" else 2), {"fp32": 4, "bf16": 2, None: 0}[c["res"]]
    rows, train = B * T * D, c["form"] == "train"
    if c["op"] == "mlp":
        return {"bytes": (2 * rows + 3 * D * F) * e * (2 if train else 1), "flops": rows * F * (18 if train else 6)}
    if c["op"] == "drop":
        return {"bytes": 2 * rows * e * (2 if train else 1), "flops": 20 * rows * (2 if train else 1)}
    params, random = 4 * D * (2 if c["bias"] else 1), 20 if c["p"] else 0
    if train:
        return {"bytes": rows * 4 * (e + r) + 2 * params, "flops": (22 + 2 * random) * rows}
    return {"bytes": rows * 2 * (e + r) + params, "flops": (8 + random) * rows}
