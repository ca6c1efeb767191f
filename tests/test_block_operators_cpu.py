"""Operators around the recurrences without a GPU: their plain forms against differentiation and differences, and every call that
they refuse before anything is launched."""
import ctypes as C
import math

import pytest
import torch

from oracle import block_oracle as bo


def _scan_inputs(gen, bt, T, ch, N, G=1):
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    return dict(u=r(bt, T, ch), delta=r(bt, T, ch), A=-torch.rand(ch, N, generator=gen, dtype=torch.float64) * 2, B=r(bt, T, G, N),
                C=r(bt, T, G, N), D=r(ch), z=r(bt, T, ch), delta_bias=r(ch) - 1)


@pytest.mark.parametrize("softplus,G,cu", [(True, 2, None), (False, 1, [0, 3, 3, 7])])
def test_scan_formulas_are_the_gradients(softplus, G, cu):
    gen = torch.Generator().manual_seed(1)
    bt, T, ch, N = (2, 7, 4, 3) if cu is None else (1, 7, 4, 3)
    seqs = bt if cu is None else len(cu) - 1
    inp = _scan_inputs(gen, bt, T, ch, N, G)
    inp["delta_bias"] += 0 if softplus else 1.5
    init = torch.randn(seqs, ch, N, generator=gen, dtype=torch.float64)
    dy, df = torch.randn(bt, T, ch, generator=gen, dtype=torch.float64), torch.randn(seqs, ch, N, generator=gen, dtype=torch.float64)
    leaves = {k: v.clone().requires_grad_(True) for k, v in inp.items()}
    i0 = init.clone().requires_grad_(True)

    def loss(kw, i):
        y, fin, _, _ = bo.scan(**kw, softplus=softplus, init=i, cu=cu)
        return (y * dy).sum() + (fin * df).sum()

    auto = torch.autograd.grad(loss(leaves, i0), list(leaves.values()) + [i0])
    got = bo.scan_grads(dy, **inp, softplus=softplus, init=init, cu=cu, d_final=df)
    names = ["du", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "d_init"]
    for n, a in zip(names, auto):
        assert torch.allclose(got[n], a, rtol=1e-10, atol=1e-10), n
    # and differences along a direction
    v = {k: torch.randn(t.shape, generator=gen, dtype=torch.float64) for k, t in inp.items()}
    h = 1e-5
    d = (loss({k: inp[k] + h * v[k] for k in inp}, init) - loss({k: inp[k] - h * v[k] for k in inp}, init)) / (2 * h)
    by_grad = sum((got["d" + k] * v[k]).sum() for k in inp)
    assert abs(d - by_grad) <= 1e-6 * (1 + abs(by_grad))


def test_conv_form_is_a_convolution_and_hands_its_state_on():
    gen = torch.Generator().manual_seed(2)
    x, w, b = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((2, 9, 3), (3, 4), (3,)))
    y, fin = bo.conv(x, w, b, silu=False)
    ref = torch.nn.functional.conv1d(torch.nn.functional.pad(x.transpose(1, 2), (3, 0)), w.unsqueeze(1), b, groups=3).transpose(1, 2)
    assert torch.allclose(y, ref)
    assert torch.equal(fin, x[:, -4:].transpose(1, 2))
    first, state = bo.conv(x[:, :2], w, b, silu=False)
    rest, _ = bo.conv(x[:, 2:], w, b, silu=False, init=state)
    assert torch.allclose(torch.cat([first, rest], 1), y)


@pytest.fixture(scope="module")
def L():
    from palimpsa_amd import _lib

    _lib.load()
    return _lib


P = C.c_void_p(0x1000)


def _norm_dims(L, **kw):
    return L.PalNormDims(**{**dict(rows=4, x_stride=64, res_stride=64, dim=64, dtype=1, res_dtype=1, weight_dtype=0, group=0, eps=1e-5),
                            **kw})


def test_norm_entry_points_refuse(L):
    lib = L.load()
    t = L.PalNormTensors(x=P, residual=P, weight=P, residual_out=P, y=P)
    fwd = lambda d, t=t: lib.pal_residual_norm_fwd(d, t, None)  # noqa: E731
    assert fwd(None) == L.PAL_E_NULL and fwd(_norm_dims(L), None) == L.PAL_E_NULL
    for kw in (dict(rows=0), dict(dim=0), dict(dim=16385, x_stride=16385, res_stride=16385), dict(x_stride=63), dict(res_stride=8), dict(group=48),
               dict(group=16), dict(group=512, dim=512, x_stride=512, res_stride=512), dict(group=128), dict(eps=-1.0), dict(eps=math.nan)):
        assert fwd(_norm_dims(L, **kw)) == L.PAL_E_DIM, kw
    for kw in (dict(dtype=2), dict(res_dtype=7), dict(weight_dtype=-1), dict(dtype=0, res_dtype=1)):
        assert fwd(_norm_dims(L, **kw)) == L.PAL_E_DTYPE, kw
    assert fwd(_norm_dims(L), L.PalNormTensors(x=P, weight=P, y=P)) == L.PAL_E_NULL
    bwd = lambda d, t, g, ws=P, n=1 << 20: lib.pal_residual_norm_bwd(d, t, g, ws, n, None)  # noqa: E731
    g = L.PalNormGrads(dy=P, dx=P, dweight=P)
    assert bwd(_norm_dims(L), t, None) == L.PAL_E_NULL
    assert bwd(_norm_dims(L, res_dtype=0), t, g) == L.PAL_E_NULL            # two types need two gradients
    assert bwd(_norm_dims(L), t, g, None, 0) == L.PAL_E_WORKSPACE and bwd(_norm_dims(L), t, g, P, 16) == L.PAL_E_WORKSPACE
    assert bwd(_norm_dims(L), t, g, C.c_void_p(0x1004)) == L.PAL_E_ALIGN
    assert lib.pal_residual_norm_bwd_workspace_bytes(_norm_dims(L)) == 4 * 64 and lib.pal_residual_norm_bwd_workspace_bytes(_norm_dims(L, dim=0)) == 0


def _conv_dims(L, **kw):
    return L.PalConvDims(**{**dict(batch=2, seq_len=16, n_seqs=2, channels=8, width=4, total_chunks=0, dtype=1, weight_dtype=0, silu=1, flags=0,
                                   x_batch_stride=128, x_token_stride=8), **kw})


def test_conv_entry_points_refuse(L):
    lib = L.load()
    t = dict(x=P, weight=P, bias=P, y=P)
    fwd = lambda d, **kw: lib.pal_short_conv_fwd(d, L.PalConvTensors(**{**t, **kw}), None)  # noqa: E731
    assert lib.pal_short_conv_fwd(None, None, None) == L.PAL_E_NULL
    for kw in (dict(batch=0), dict(seq_len=0), dict(n_seqs=0), dict(n_seqs=3), dict(channels=0), dict(width=1), dict(width=9),
               dict(x_token_stride=7), dict(x_batch_stride=-1), dict(batch=1 << 16, seq_len=1 << 15)):
        assert fwd(_conv_dims(L, **kw)) == L.PAL_E_DIM, kw
    assert fwd(_conv_dims(L, dtype=3)) == L.PAL_E_DTYPE and fwd(_conv_dims(L, weight_dtype=9)) == L.PAL_E_DTYPE
    assert fwd(_conv_dims(L), x=None) == L.PAL_E_NULL
    packed = dict(batch=1, flags=L.PAL_FLAG_VARLEN, n_seqs=3, total_chunks=2)
    assert fwd(_conv_dims(L, flags=L.PAL_FLAG_VARLEN), cu_seqlens=P, chunk_table=P) == L.PAL_E_VARLEN_BATCH
    assert fwd(_conv_dims(L, **packed)) == L.PAL_E_CU_SEQLENS and fwd(_conv_dims(L), cu_seqlens=P) == L.PAL_E_CU_SEQLENS
    assert fwd(_conv_dims(L, **packed), cu_seqlens=P) == L.PAL_E_NULL
    assert fwd(_conv_dims(L, **{**packed, "total_chunks": 4}), cu_seqlens=P, chunk_table=P) == L.PAL_E_CHUNK
    assert fwd(_conv_dims(L, flags=L.PAL_FLAG_HAS_INIT)) == L.PAL_E_STATE and fwd(_conv_dims(L), init=P) == L.PAL_E_STATE
    assert fwd(_conv_dims(L, flags=L.PAL_FLAG_STORE_FINAL)) == L.PAL_E_STATE and fwd(_conv_dims(L), final_=P) == L.PAL_E_STATE
    g = dict(dy=P, dx=P, dweight=P, dbias=P)
    bwd = lambda g, ws=P, n=1 << 20, **kw: lib.pal_short_conv_bwd(_conv_dims(L), L.PalConvTensors(**{**t, **kw}), L.PalConvGrads(**g), ws, n, None)  # noqa: E731
    assert bwd({**g, "dbias": None}) == L.PAL_E_NULL and bwd(g, bias=None) == L.PAL_E_NULL
    assert bwd({**g, "d_init": P}) == L.PAL_E_STATE
    assert bwd(g, None, 0) == L.PAL_E_WORKSPACE and bwd(g, P, 8) == L.PAL_E_WORKSPACE
    step = lambda d, **kw: lib.pal_short_conv_step(d, L.PalConvTensors(**{**t, **kw}), None)  # noqa: E731
    assert step(_conv_dims(L)) == L.PAL_E_STATE and step(_conv_dims(L, n_seqs=1), final_=P) == L.PAL_E_DIM
    assert step(_conv_dims(L, flags=L.PAL_FLAG_VARLEN), final_=P) == L.PAL_E_VARLEN_BATCH


def _scan_dims(L, **kw):
    s = {n + x: v for n in ("u", "delta", "z", "B", "C") for x, v in (("_batch", 1024), ("_token", 64))}
    return L.PalScanDims(**{**dict(batch=2, seq_len=16, n_seqs=2, channels=64, state=16, groups=1, dtype=1, softplus=1, flags=0), **s, **kw})


def test_scan_entry_points_refuse(L):
    lib = L.load()
    t = dict(u=P, delta=P, A=P, B=P, C=P, y=P)
    fwd = lambda d, ws=None, n=0, **kw: lib.pal_scan_fwd(d, L.PalScanTensors(**{**t, **kw}), ws, n, None)  # noqa: E731
    assert lib.pal_scan_fwd(None, None, None, 0, None) == L.PAL_E_NULL
    for kw in (dict(batch=0), dict(seq_len=0), dict(n_seqs=1), dict(channels=0), dict(groups=0), dict(groups=3), dict(state=0), dict(state=65),
               dict(u_token=-1), dict(batch=65536, n_seqs=65536)):
        assert fwd(_scan_dims(L, **kw)) == L.PAL_E_DIM, kw
    assert fwd(_scan_dims(L, dtype=2)) == L.PAL_E_DTYPE
    assert fwd(_scan_dims(L, flags=L.PAL_FLAG_VARLEN), cu_seqlens=P) == L.PAL_E_VARLEN_BATCH
    assert fwd(_scan_dims(L), cu_seqlens=P) == L.PAL_E_CU_SEQLENS
    assert fwd(_scan_dims(L, flags=L.PAL_FLAG_HAS_INIT)) == L.PAL_E_STATE and fwd(_scan_dims(L), init=P) == L.PAL_E_STATE
    assert fwd(_scan_dims(L), final_=P) == L.PAL_E_STATE
    assert fwd(_scan_dims(L), A=C.c_void_p(0x1008)) == L.PAL_E_ALIGN
    both = L.PAL_FLAG_HAS_INIT | L.PAL_FLAG_STORE_FINAL      # of a packed batch one segment reads what another writes
    assert fwd(_scan_dims(L, batch=1, flags=L.PAL_FLAG_VARLEN | both), cu_seqlens=P, init=P, final_=P) == L.PAL_E_STATE
    assert fwd(_scan_dims(L, u_token=1 << 24)) == L.PAL_E_DIM
    assert fwd(_scan_dims(L, channels=1 << 21, groups=1 << 21)) == L.PAL_E_DIM
    assert fwd(_scan_dims(L), y=None) == L.PAL_E_NULL and fwd(_scan_dims(L), C=None) == L.PAL_E_NULL
    long = dict(batch=1, n_seqs=1, seq_len=100000)
    need = lib.pal_scan_fwd_workspace_bytes(_scan_dims(L, **long))
    assert need > 0 and lib.pal_scan_fwd_workspace_bytes(_scan_dims(L)) == 0
    assert fwd(_scan_dims(L, **long)) == L.PAL_E_WORKSPACE and fwd(_scan_dims(L, **long), P, need - 1) == L.PAL_E_WORKSPACE
    assert lib.pal_scan_checkpoint_bytes(_scan_dims(L)) == 2 * 2 * 4096 and lib.pal_scan_checkpoint_bytes(_scan_dims(L, state=99)) == 0
    g = dict(dy=P, du=P, ddelta=P, dA=P, dB=P, dC=P)
    bwd = lambda g, ws=P, n=1 << 30, **kw: lib.pal_scan_bwd(_scan_dims(L), L.PalScanTensors(**{**t, "checkpoints": P, **kw}), L.PalScanGrads(**g), ws, n, None)  # noqa: E731
    assert bwd(g, checkpoints=None) == L.PAL_E_NULL and bwd({**g, "dA": None}) == L.PAL_E_NULL
    for x, dx in (("D", "dD"), ("z", "dz"), ("delta_bias", "ddelta_bias")):
        assert bwd(g, **{x: P}) == L.PAL_E_NULL and bwd({**g, dx: P}) == L.PAL_E_NULL
    assert bwd({**g, "d_init": P}) == L.PAL_E_STATE
    assert bwd(g, None, 0) == L.PAL_E_WORKSPACE and bwd(g, P, 64) == L.PAL_E_WORKSPACE


def test_entry_points_run_on_a_gpu_only():
    from palimpsa_amd.ops.layer_glue import residual_rms_norm, residual_rms_norm_fp8
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step

    x, w = torch.randn(1, 4, 8), torch.randn(8, 4)
    bc, A = torch.randn(1, 4, 2), -torch.rand(8, 2)
    for call in (lambda: short_conv(x, w), lambda: short_conv_step(x, torch.zeros(1, 8, 4), w), lambda: selective_scan(x, x, A, bc, bc),
                 lambda: selective_scan_step(x, torch.zeros(1, 8, 2), x, A, bc, bc), lambda: residual_rms_norm(x, None, torch.ones(8)),
                 lambda: residual_rms_norm_fp8(x, x, torch.ones(8))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_conv_passes_of_more_threads_than_a_launch_holds_are_refused(L):
    """2^32 threads: refused as a size, before a launch that the runtime would turn down."""
    lib = L.load()
    t = L.PalConvTensors(x=P, weight=P, y=P, final_=P)
    step = _conv_dims(L, batch=1 << 22, n_seqs=1 << 22, seq_len=1, channels=1 << 10, x_token_stride=1 << 10, x_batch_stride=1 << 10)
    assert lib.pal_short_conv_step(step, t, None) == L.PAL_E_DIM
    many = _conv_dims(L, batch=1 << 27, n_seqs=1 << 27, seq_len=1, channels=4, x_token_stride=4, x_batch_stride=4)
    t = L.PalConvTensors(x=P, weight=P, y=P)
    need = lib.pal_short_conv_bwd_workspace_bytes(many)
    assert lib.pal_short_conv_bwd(many, t, L.PalConvGrads(dy=P, dx=P, dweight=P), P, need, None) == L.PAL_E_DIM


def test_scan_backward_of_more_tiles_than_its_sums_hold_is_refused(L):
    """A million groups of one channel: the last launch would have 5 x 2^30 threads."""
    lib = L.load()
    n = 1 << 20
    d = L.PalScanDims(batch=1, seq_len=8, n_seqs=1, channels=n, state=8, groups=n, dtype=1, softplus=1, flags=0,
                      **{x + "_batch": 0 for x in ("u", "delta", "z", "B", "C")}, u_token=n, delta_token=n, z_token=n, B_token=8 * n, C_token=8 * n)
    t = L.PalScanTensors(u=P, delta=P, A=P, B=P, C=P, y=P, checkpoints=P)
    g = L.PalScanGrads(dy=P, du=P, ddelta=P, dA=P, dB=P, dC=P)
    assert lib.pal_scan_bwd(d, t, g, P, lib.pal_scan_bwd_workspace_bytes(d), None) == L.PAL_E_DIM
