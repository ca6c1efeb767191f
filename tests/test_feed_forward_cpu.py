"""The feed-forward half's operators without a GPU: their plain forms against differentiation, differences and known answers, and every call that
they refuse before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import feed_forward_oracle as fo

P = C.c_void_p(0x1000)


@pytest.fixture(scope="module")
def L():
    from palimpsa_amd import _lib, build
    import os
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    _lib.load()
    return _lib


def test_philox_known_answers():
    """The authors' test vectors (Random123): zero, all ones, digits of pi."""
    ones = 0xFFFFFFFF
    pi, key = (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)
    hexes = lambda c, k, r: [format(int(w), "08x") for w in fo.philox(np.array([c], dtype=np.uint64), k, r)[0]]  # noqa: E731
    assert hexes((0, 0, 0, 0), (0, 0), 10) == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]
    assert hexes((ones,) * 4, (ones, ones), 10) == ["408f276d", "41c83b0e", "a20bc7c6", "6d5451fd"]
    assert hexes(pi, key, 10) == ["d16cfe09", "94fdcceb", "5001e420", "24126ea1"]
    assert hexes((0, 0, 0, 0), (0, 0), 7) == ["5f6fb709", "0d893f64", "4f121f81", "4f730a48"]


def test_kept_share_and_independence():
    n = 400 * 1001
    for p in (0.1, 0.5, 0.9):
        k = fo.kept((400, 1001), p, 7).double()
        assert abs(k.mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    a, b, c = (fo.kept((400, 1001), 0.5, s, t) for s, t in ((7, 0), (8, 0), (7, 1)))
    for x in (b, c):
        assert abs((a == x).double().mean().item() - 0.5) < 5 * 0.5 / n ** 0.5
    assert torch.equal(fo.kept((5, 9), 0.5, 7)[3:4], fo.kept((400, 9), 0.5, 7)[3:4])          # by place alone
    assert fo.kept((3, 5), 0.0, 1).all() and torch.equal(fo.kept((3, 5), 0.3, -1), fo.kept((3, 5), 0.3, 2 ** 64 - 1))


def _close_to_differences(loss, leaves, grads, gen):
    v = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in leaves]
    h = 1e-6
    with torch.no_grad():
        d = (loss(*[t + h * u for t, u in zip(leaves, v)]) - loss(*[t - h * u for t, u in zip(leaves, v)])) / (2 * h)
    by = sum((g * u).sum() for g, u in zip(grads, v))
    assert abs(d - by) <= 1e-6 * (1 + abs(by))


def test_layer_norm_formulas_are_the_gradients():
    gen = torch.Generator().manual_seed(1)
    s, w, b, dy = (torch.randn(*n, generator=gen, dtype=torch.float64) for n in ((5, 13), (13,), (13,), (5, 13)))
    loss = lambda s, w, b: (fo.layer_norm(s, w, b)[0] * dy).sum()  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (s, w, b)]
    auto = torch.autograd.grad(loss(*leaves), leaves)
    y, hat, r = fo.layer_norm(s, w, b)
    assert torch.allclose(y, torch.nn.functional.layer_norm(s, (13,), w, b, 1e-5), rtol=1e-12)
    got = fo.layer_norm_grads(dy, hat, r, w)
    for g, a in zip(got, auto):
        assert torch.allclose(g, a, rtol=1e-10, atol=1e-12)
    _close_to_differences(loss, leaves, got, gen)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_gated_mlp_formulas_are_the_gradients(act):
    gen = torch.Generator().manual_seed(2)
    x, wg, wu, wd, dy = (torch.randn(*n, generator=gen, dtype=torch.float64) for n in ((6, 5), (7, 5), (7, 5), (4, 7), (6, 4)))
    loss = lambda *t: (fo.gated_mlp(*t, act)[0] * dy).sum()  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    auto = torch.autograd.grad(loss(*leaves), leaves)
    got = fo.gated_mlp_grads(dy, x, wg, wu, wd, act)
    for g, a in zip(got, auto):
        assert torch.allclose(g, a, rtol=1e-10, atol=1e-12)
    _close_to_differences(loss, leaves, got, gen)
    z = torch.linspace(-6, 6, 41, dtype=torch.float64)
    ref = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
           "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act]
    assert torch.allclose(fo.activation(act, z)[0], ref(z), rtol=1e-9, atol=1e-12)


# --------------------------------------------------------------------------------------------------------- the C ABI
def _mlp_dims(L, **kw):
    return L.PalMlpDims(**{**dict(rows=64, x_stride=64, dim=64, hidden=128, out_dim=64, dtype=1, activation=0), **kw})


def test_gated_mlp_entry_points_refuse(L):
    lib = L.load()
    t = dict(x=P, w_gate=P, w_up=P, w_down=P, y=P)
    big = 1 << 40
    fwd = lambda d, ws=P, n=big, **kw: lib.pal_gated_mlp_fwd(d, L.PalMlpTensors(**{**t, **kw}), ws, n, None)  # noqa: E731
    g = dict(dy=P, dx=P, dw_gate=P, dw_up=P, dw_down=P)
    bwd = lambda d, ws=P, n=big, gr=g, **kw: lib.pal_gated_mlp_bwd(d, L.PalMlpTensors(**{**t, "kept": P, **kw}), L.PalMlpGrads(**gr), ws, n, None)  # noqa: E731
    assert lib.pal_gated_mlp_fwd(None, None, None, 0, None) == L.PAL_E_NULL
    for call in (fwd, bwd):
        for kw in (dict(rows=0), dict(rows=(1 << 30) + 1), dict(dim=0), dict(dim=60), dict(hidden=4), dict(hidden=-8), dict(out_dim=12), dict(x_stride=56),
                   dict(x_stride=68), dict(x_stride=(1 << 20) + 8), dict(activation=4), dict(activation=-1), dict(dim=(1 << 20) + 8)):
            assert call(_mlp_dims(L, **kw)) == L.PAL_E_DIM, kw
        assert call(_mlp_dims(L, dtype=2)) == L.PAL_E_DTYPE
        for name in ("x", "w_gate", "w_up", "w_down"):
            assert call(_mlp_dims(L), **{name: None}) == L.PAL_E_NULL
            assert call(_mlp_dims(L), **{name: C.c_void_p(0x1008)}) == L.PAL_E_ALIGN
        assert call(_mlp_dims(L), kept=C.c_void_p(0x1004)) == L.PAL_E_ALIGN
        assert call(_mlp_dims(L), None) == L.PAL_E_WORKSPACE and call(_mlp_dims(L), P, 8) == L.PAL_E_WORKSPACE
        assert call(_mlp_dims(L), C.c_void_p(0x1008)) == L.PAL_E_ALIGN
    assert fwd(_mlp_dims(L), y=None) == L.PAL_E_NULL
    assert bwd(_mlp_dims(L), kept=None) == L.PAL_E_NULL and bwd(_mlp_dims(L), gr={**g, "dy": None}) == L.PAL_E_NULL
    assert bwd(_mlp_dims(L), gr={**g, "dx": C.c_void_p(0x1008)}) == L.PAL_E_ALIGN


def test_gated_mlp_sizes(L):
    lib = L.load()
    assert lib.pal_gated_mlp_kept_bytes(_mlp_dims(L)) > 0 and lib.pal_gated_mlp_kept_bytes(_mlp_dims(L, dim=5)) == 0
    some = L.PalMlpGrads(dy=P, dw_up=P)
    assert lib.pal_gated_mlp_bwd_workspace_bytes(_mlp_dims(L), some) >= 2 * 64 * 128 * 2 and lib.pal_gated_mlp_bwd_workspace_bytes(_mlp_dims(L, dim=5), some) == 0
    assert lib.pal_gated_mlp_bwd_workspace_bytes(_mlp_dims(L), None) == 0
    assert lib.pal_gated_mlp_fwd_workspace_bytes(_mlp_dims(L, hidden=5), 0) == 0
    # rows of h an odd number of 128-byte lines apart, three arrays of them kept
    assert lib.pal_gated_mlp_kept_bytes(_mlp_dims(L, rows=16, hidden=2048)) == 3 * 16 * (4096 + 128)
    # up to sixteen rows of bf16 have h in two parts, of which the first is kept
    for dtype, keeps, n in ((1, 0, 2), (1, 1, 1), (0, 0, 1), (0, 1, 0)):
        line = 2048 * (2 if dtype else 4) + 128
        assert lib.pal_gated_mlp_fwd_workspace_bytes(_mlp_dims(L, rows=16, hidden=2048, dtype=dtype), keeps) == n * 16 * line


def _norm_dims(L, drop=None, **kw):
    d = L.PalLayerNormDims(**{**dict(rows=4, x_stride=64, res_stride=64, dim=64, dtype=1, res_dtype=1, weight_dtype=0, eps=1e-5), **kw})
    if drop is not None:
        d.drop = drop
    return d


def test_layer_norm_entry_points_refuse(L):
    lib = L.load()
    t = dict(x=P, residual=P, weight=P, bias=P, residual_out=P, y=P, stats=P)
    g = dict(dy=P, dresidual_out=P, dx=P, dresidual=P, dweight=P, dbias=P)
    fwd = lambda d, **kw: lib.pal_layer_norm_fwd(d, L.PalLayerNormTensors(**{**t, **kw}), None)  # noqa: E731
    bwd = lambda d, ws=P, n=1 << 40, gr=g, **kw: lib.pal_layer_norm_bwd(d, L.PalLayerNormTensors(**{**t, **kw}), L.PalLayerNormGrads(**gr), ws, n, None)  # noqa: E731
    assert lib.pal_layer_norm_fwd(None, None, None) == L.PAL_E_NULL
    for call in (fwd, bwd):
        for kw in (dict(rows=0), dict(dim=0), dict(dim=16385, x_stride=16385, res_stride=16385), dict(x_stride=63), dict(res_stride=63), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(rows=(1 << 40) + 1)):
            assert call(_norm_dims(L, **kw)) == L.PAL_E_DIM, kw
        for p in (-0.1, 1.0, 1.5, float("nan")):
            assert call(_norm_dims(L, L.PalDropout(p=p))) == L.PAL_E_DIM, p
        for kw in (dict(dtype=2), dict(res_dtype=2), dict(weight_dtype=2), dict(dtype=0, res_dtype=1)):
            assert call(_norm_dims(L, **kw)) == L.PAL_E_DTYPE, kw
        assert call(_norm_dims(L), weight=None) == L.PAL_E_NULL
        assert call(_norm_dims(L), stats=C.c_void_p(0x1004)) == L.PAL_E_ALIGN
        assert call(_norm_dims(L, res_dtype=0), residual_out=None) == L.PAL_E_NULL
        assert call(_norm_dims(L, L.PalDropout(p=0.5)), residual=None, residual_out=None) == L.PAL_E_NULL
    assert fwd(_norm_dims(L), x=None) == L.PAL_E_NULL and fwd(_norm_dims(L), y=None) == L.PAL_E_NULL
    assert fwd(_norm_dims(L), residual_out=None) == L.PAL_E_NULL                # the stream is handed on
    assert bwd(_norm_dims(L), stats=None) == L.PAL_E_NULL and bwd(_norm_dims(L), x=None, residual_out=None) == L.PAL_E_NULL
    for name in ("dx", "dweight", "dbias"):
        assert bwd(_norm_dims(L), gr={**g, name: None}) == L.PAL_E_NULL
    assert bwd(_norm_dims(L), bias=None) == L.PAL_E_NULL                        # dbias iff bias
    assert bwd(_norm_dims(L), None) == L.PAL_E_WORKSPACE and bwd(_norm_dims(L), P, 8) == L.PAL_E_WORKSPACE
    assert bwd(_norm_dims(L), C.c_void_p(0x1004)) == L.PAL_E_ALIGN
    assert lib.pal_layer_norm_bwd_workspace_bytes(_norm_dims(L)) == 2 * 64 * 4 and lib.pal_layer_norm_bwd_workspace_bytes(_norm_dims(L, dim=0)) == 0


def test_dropout_entry_point_refuses(L):
    lib = L.load()
    call = lambda p=0.5, x=P, y=P, rows=4, dim=8, stride=8, dtype=1: lib.pal_dropout(L.PalDropout(p=p), x, y, rows, dim, stride, dtype, None)  # noqa: E731
    assert lib.pal_dropout(None, P, P, 4, 8, 8, 1, None) == L.PAL_E_NULL
    assert call(x=None) == L.PAL_E_NULL and call(y=None) == L.PAL_E_NULL and call(dtype=2) == L.PAL_E_DTYPE
    for kw in (dict(rows=0), dict(dim=0), dict(dim=(1 << 30) + 1, stride=(1 << 30) + 1), dict(stride=7), dict(p=1.0), dict(p=-1e-9), dict(p=float("nan"))):
        assert call(**kw) == L.PAL_E_DIM, kw
    # entries in all are counted in 64 bits
    for rows, dim in ((1 << 40, 1 << 30), (1 << 37, 1 << 30), ((1 << 36) + 1, 1 << 10)):
        assert call(rows=rows, dim=dim, stride=dim) == L.PAL_E_DIM, (rows, dim)


def test_copy_entry_point_refuses(L):
    lib = L.load()
    ok = dict(src=P, dst=P, src_ld=9, dst_ld=16, rows=3, cols=9, dst_rows=8, dst_cols=16)

    def call(n=1, dtype=1, **kw):
        m = (L.PalMatrixCopy * 9)(*[L.PalMatrixCopy(**ok)] * 8)
        m[max(min(n, 8) - 1, 0)] = L.PalMatrixCopy(**{**ok, **kw})
        return lib.pal_copy_matrices(m, n, dtype, None)

    assert lib.pal_copy_matrices(None, 1, 1, None) == L.PAL_E_NULL
    for n in (1, 3, 8):
        assert call(n, src=None) == L.PAL_E_NULL and call(n, dst=None) == L.PAL_E_NULL
        for kw in (dict(rows=0), dict(cols=0), dict(rows=9), dict(cols=17), dict(src_ld=8), dict(dst_ld=15), dict(dst_rows=(1 << 30) + 1),
                   dict(dst_cols=(1 << 30) + 1, dst_ld=1 << 31)):
            assert call(n, **kw) == L.PAL_E_DIM, kw
    assert call(0) == L.PAL_E_DIM and call(9) == L.PAL_E_DIM and call(dtype=2) == L.PAL_E_DTYPE


# ------------------------------------------------------------------------------------------------ the Python boundary
def test_calls_that_are_refused():
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm, residual_layer_norm
    x, w, m = torch.zeros(2, 8), torch.ones(8), torch.zeros(8, 8)
    for f in (lambda: layer_norm(x, w), lambda: residual_layer_norm(x, x, w), lambda: dropout(x, 0.5, 1), lambda: gated_mlp(x, m, m, m)):
        with pytest.raises(RuntimeError, match="GPU only"):
            f()
    for p in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            residual_layer_norm(x, x, w, dropout_p=p, seed=1)
    with pytest.raises(ValueError, match="needs a seed"):
        residual_layer_norm(x, x, w, dropout_p=0.5)
    for seed in (1.5, None, 1 << 64, -(1 << 63) - 1, torch.zeros(1), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="seed"):
            residual_layer_norm(x, x, w, dropout_p=0.5, seed=seed)
    for site in (-1, 1 << 32, 0.0):
        with pytest.raises(ValueError, match="site"):
            residual_layer_norm(x, x, w, dropout_p=0.5, seed=1, site=site)


def test_shapes_that_are_refused():
    from palimpsa_amd.ops import gated_mlp as gm
    m = torch.zeros
    ok = (m(3, 8), m(16, 8), m(16, 8), m(4, 16))
    gm._check(*ok, "silu")
    with pytest.raises(ValueError, match="activation"):
        gm._check(*ok, "swish")
    for i, t in ((0, m(3, 7)), (1, m(16, 9)), (2, m(15, 8)), (3, m(4, 15)), (3, m(16)), (1, m(16, 8, 1)), (0, m(()))):
        with pytest.raises(ValueError, match="expected x"):
            gm._check(*[t if j == i else u for j, u in enumerate(ok)], "silu")
    with pytest.raises(ValueError, match="dims must be"):
        gm._check(m(3, 8), m(0, 8), m(0, 8), m(4, 0), "silu")
