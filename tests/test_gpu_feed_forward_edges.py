"""Edges of the feed-forward half's operators on the GPU: layouts, types, missing gradients, not finite numbers, graphs, streams, memory around the
results, far offsets, and the operators together as a block uses them."""
import ctypes as C

import pytest
import torch

from oracle import feed_forward_oracle as fo
from tests import feed_forward_bounds as fb
from tests import helpers as hp
from tests.test_gpu_gated_mlp import make

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _randn(dev, *shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


# ------------------------------------------------------------------------------------------------------------- layouts
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [7, 200])
def test_layouts_of_the_block_give_the_same_bits(gpu_device, dtype, M):
    from palimpsa_amd.ops.gated_mlp import _gated_mlp, gated_mlp
    x, wg, wu, wd, dy = make(gpu_device, M, 64, 96, 64, dtype)

    def run(f, *a, dy=dy):
        leaves = [t.detach().requires_grad_(True) for t in a]
        y = f(*leaves, "silu")
        return [y] + list(torch.autograd.grad(y, leaves, dy))

    want = run(gated_mlp, x, wg, wu, wd)
    wide = _randn(gpu_device, M, 128, seed=9, dtype=dtype)
    wide[:, 40:104] = x
    both = torch.cat([wg, wu])
    off = torch.empty(M * 64 + 3, dtype=dtype, device=gpu_device)[3:].view(M, 64)
    off.copy_(x)
    variants = {
        "a slice of wider rows": (wide[:, 40:104], wg, wu, wd),
        "rows off by three elements": (off, wg, wu, wd),
        "columns first": (x.t().contiguous().t(), wg.t().contiguous().t(), wu.t().contiguous().t(), wd.t().contiguous().t()),
        "halves of one matrix": (x, both[:96], both[96:], wd),
    }
    for name, a in variants.items():
        for got, ref in zip(run(gated_mlp, *a), want):
            assert torch.equal(got, ref), name
    for got, ref in zip(run(_gated_mlp, x, wg, wu, wd), want):
        assert torch.equal(got, ref), "Python route"
    for got, ref in zip(run(gated_mlp, x, wg, wu, wd, dy=dy.t().contiguous().t()), want):
        assert torch.equal(got, ref), "gradient's layout"
    for got, ref in zip(run(gated_mlp, x.view(1, M, 1, 64), wg, wu, wd, dy=dy.view(1, M, 1, 64)), want):
        assert torch.equal(got.reshape(ref.shape), ref)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,D,Fh,Do", [(7, 61, 97, 3), (200, 64, 97, 64), (130, 61, 96, 72), (1, 8, 9, 5), (70, 515, 40, 1027)])
def test_odd_layouts_of_the_block_give_the_same_bits(gpu_device, dtype, M, D, Fh, Do):
    from palimpsa_amd import _lib as L
    from palimpsa_amd.ops.gated_mlp import _gated_mlp, gated_mlp
    x, wg, wu, wd, dy = make(gpu_device, M, D, Fh, Do, dtype)

    def run(f, *a):
        leaves = [t.detach().requires_grad_(True) for t in a]
        y = f(*leaves, "silu")
        with torch.no_grad():
            assert torch.equal(f(*leaves, "silu"), y)
        one = torch.autograd.grad(f(*leaves, "silu"), leaves[2:3], dy)[0]      # a part of the gradients
        grads = torch.autograd.grad(y, leaves, dy)
        assert torch.equal(one, grads[2])
        return [y] + list(grads)

    with torch.no_grad():
        assert L.host().gated_mlp(x, wg, wu, wd, 0) is not None
    want = run(_gated_mlp, x, wg, wu, wd)
    wide = _randn(gpu_device, M, D + 13, seed=9, dtype=dtype)
    wide[:, 5:5 + D] = x
    off = lambda t: torch.empty(t.numel() + 3, dtype=dtype, device=t.device)[3:].view(t.shape).copy_(t)  # noqa: E731
    for a in ((x, wg, wu, wd), (wide[:, 5:5 + D], wg, wu, wd), (off(x), off(wg), off(wu), off(wd))):
        for got, ref in zip(run(gated_mlp, *a), want):
            assert got.shape == ref.shape and torch.equal(got, ref)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_copies_of_matrices(gpu_device, dtype):
    """Several at a time, rows and columns behind them zero, at odd addresses; nothing around them is written."""
    from palimpsa_amd import _lib as L
    sizes = [(1, 1, 1, 1), (3, 5, 8, 8), (130, 771, 136, 776), (9, 8, 9, 8), (1000, 17, 1000, 19), (2, 5000, 2, 5000)]
    src = [_randn(gpu_device, r, c + 3, seed=i, dtype=dtype) for i, (r, c, _, _) in enumerate(sizes)]
    room = [torch.full((r8 * (c8 + 2) + 6,), 7.0, dtype=dtype, device=gpu_device) for _, _, r8, c8 in sizes]
    es = src[0].element_size()
    m = (L.PalMatrixCopy * len(sizes))(*[
        L.PalMatrixCopy(src=s.data_ptr() + es, dst=d.data_ptr() + 3 * es, src_ld=c + 3, dst_ld=c8 + 2, rows=r, cols=c, dst_rows=r8, dst_cols=c8)
        for s, d, (r, c, r8, c8) in zip(src, room, sizes)])
    assert L.load().pal_copy_matrices(m, len(sizes), int(dtype == BF), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    for s, d, (r, c, r8, c8) in zip(src, room, sizes):
        want = torch.full_like(d, 7.0)
        inner = want[3:3 + r8 * (c8 + 2)].view(r8, c8 + 2)
        inner[:, :c8] = 0
        inner[:r, :c] = s[:, 1:1 + c]
        assert torch.equal(d, want)


def test_layouts_of_the_norm_and_dropout_give_the_same_bits(gpu_device):
    from palimpsa_amd.ops.layer_glue import _dropout, _layer_norm, dropout, layer_norm, residual_layer_norm
    x, res, w, b, dy, dr = (_randn(gpu_device, *s, seed=i, dtype=BF) for i, s in enumerate(((6, 5, 100), (6, 5, 100), (100,), (100,), (6, 5, 100), (6, 5, 100))))

    def run(f, *a):
        leaves = [t.detach().requires_grad_(True) for t in a]
        out = f(*leaves)
        out = list(out) if isinstance(out, tuple) else [out]
        return out + list(torch.autograd.grad(out, leaves, [dy, dr][:len(out)]))

    fused = lambda x, r, w, b: residual_layer_norm(x, r, w, b, dropout_p=0.2, seed=5, site=2)  # noqa: E731
    route = lambda x, r, w, b: _layer_norm(x, r, w, b, 1e-5, False, True, 0.2, 5, None, 2)  # noqa: E731
    want = run(fused, x, res, w, b)
    for f, a in ((route, (x, res, w, b)), (fused, (torch.cat([x, x], 2)[..., :100], torch.cat([res, res], 2)[..., 100:], w, b)),
                 (fused, (x.transpose(0, 1).contiguous().transpose(0, 1), res, w, b)), (fused, (x, res, w, b.float()))):
        for i, (got, ref) in enumerate(zip(run(f, *a), want)):
            assert torch.equal(got.to(ref.dtype), ref), i       # (a bias in fp32 has its gradient in fp32)
    want = run(layer_norm, x, w, b)
    for f, a in ((lambda x, w, b: _layer_norm(x, None, w, b, 1e-5, False, False, 0.0, 0, None, 0), (x, w, b)), (layer_norm, (torch.cat([x, x], 2)[..., 100:], w, b))):
        for got, ref in zip(run(f, *a), want):
            assert torch.equal(got, ref)
    want = run(lambda t: dropout(t, 0.3, 11), x)
    for f, a in ((lambda t: _dropout(t, 0.3, 11, 0), x), (lambda t: dropout(t, 0.3, 11), torch.cat([x, x], 2)[..., 100:]),
                 (lambda t: dropout(t, 0.3, torch.tensor(11, device=gpu_device)), x), (lambda t: dropout(t, 0.3, torch.tensor([11], device=gpu_device)), x),
                 (lambda t: dropout(t.reshape(30, 100), 0.3, 11).reshape(t.shape), x)):
        for got, ref in zip(run(f, a), want):
            assert torch.equal(got, ref)


def test_other_types(gpu_device):
    """fp16 is computed from fp32 and rounded; so is anything that mixes types."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm, residual_layer_norm
    dev, H = gpu_device, torch.float16
    x, wg, wu, wd, dy = make(dev, 33, 40, 48, 24, H)
    for inp in ((x, wg, wu, wd), (x, wg.float(), wu.float(), wd.float()), (x.to(BF), wg.to(BF), wu.to(BF), wd.to(BF).float())):
        leaves = [t.requires_grad_(True) for t in inp]
        y = gated_mlp(*leaves)
        grads = torch.autograd.grad(y, leaves, dy.to(y.dtype))
        wide = [t.detach().float().requires_grad_(True) for t in inp]
        ref = gated_mlp(*wide)
        rgrads = torch.autograd.grad(ref, wide, dy.to(y.dtype).float())
        assert y.dtype == inp[0].dtype and torch.equal(y, ref.to(y.dtype))
        for g, r, t in zip(grads, rgrads, inp):
            assert g.dtype == t.dtype and torch.equal(g, r.to(t.dtype))
    h = _randn(dev, 9, 70, dtype=H)
    w = _randn(dev, 70, seed=1)
    assert torch.equal(layer_norm(h, w), layer_norm(h.float(), w).to(H)) and torch.equal(dropout(h, 0.5, 3), dropout(h.float(), 0.5, 3).to(H))
    y, s = residual_layer_norm(h, h, w)
    y2, s2 = residual_layer_norm(h.float(), h.float(), w)
    assert s.dtype == F32 and torch.equal(s, s2) and torch.equal(y, y2.to(H))


def test_gradients_that_are_not_wanted(gpu_device):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    *inp, dy = make(gpu_device, 300, 64, 128, 72, BF)
    leaves = [t.clone().requires_grad_(True) for t in inp]
    want = torch.autograd.grad(gated_mlp(*leaves), leaves, dy)
    for mask in range(1, 16):
        some = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(inp)]
        got = torch.autograd.grad(gated_mlp(*some), [t for t in some if t.requires_grad], dy)
        for g, r in zip(got, [w for i, w in enumerate(want) if mask >> i & 1]):
            # (another set of products may be cut into other shares of k: the rounding of bf16 sums at most)
            assert (g.float() - r.float()).abs().max() <= 2 ** -7 * r.float().abs().max()


@pytest.mark.parametrize("M,D,F", [(9, 64, 64), (130, 61, 61)])
def test_one_tensor_in_two_places(gpu_device, M, D, F):
    """Gate and up projection shared, down tied to both, and a stream that is added to itself: gradients are sums over the places."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import residual_layer_norm
    x, w, _, _, dy = make(gpu_device, M, D, F, D, F32)
    leaf = w.clone().requires_grad_(True)
    apart = [w.clone().requires_grad_(True) for _ in range(3)]
    y = gated_mlp(x, leaf, leaf, leaf)
    z = gated_mlp(x, *apart)
    assert torch.equal(y, z)
    (g,) = torch.autograd.grad(y, [leaf], dy)
    parts = torch.autograd.grad(z, apart, dy)
    want = sum(t.double() for t in parts)
    assert ((g - want).abs() <= 3 * 2.0 ** -24 * sum(t.double().abs() for t in parts)).all()      # two additions in fp32, in any order
    nw = _randn(gpu_device, D, seed=3)
    for p in (0.0, 0.5):
        leaf = x.clone().requires_grad_(True)
        two = [x.clone().requires_grad_(True) for _ in range(2)]
        a = residual_layer_norm(leaf, leaf, nw, dropout_p=p, seed=4)
        b = residual_layer_norm(*two, nw, dropout_p=p, seed=4)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        (g,) = torch.autograd.grad(a, [leaf], (dy, dy))
        d = torch.autograd.grad(b, two, (dy, dy))
        assert torch.equal(g, d[0] + d[1])


def test_no_rows_and_refusals(gpu_device):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm, residual_layer_norm
    x, wg, wu, wd, _ = make(gpu_device, 4, 16, 24, 8, BF)
    leaves = [t.clone().requires_grad_(True) for t in (x[:0], wg, wu, wd)]
    y = gated_mlp(*leaves)
    assert y.shape == (0, 8)
    for g, t in zip(torch.autograd.grad(y, leaves, y.detach()), leaves):
        assert g.shape == t.shape and not g.any()
    assert dropout(x[:0], 0.5, 1).shape == (0, 16) and dropout(torch.ones((), device=gpu_device), 0.0, 1).shape == ()
    with pytest.raises(ValueError, match="at least one row"):
        layer_norm(x[:0], wg[0])
    with pytest.raises(ValueError, match="up to 16384"):
        layer_norm(_randn(gpu_device, 2, 16385), _randn(gpu_device, 16385))
    with pytest.raises(ValueError, match="shape of x"):
        residual_layer_norm(x, x[:2], wg[0])
    with pytest.raises(ValueError, match=r"must be \[16\]"):
        layer_norm(x, wg[0], wg[0][:8])
    with pytest.raises(ValueError, match="negative"):
        layer_norm(x, wg[0], eps=-1.0)
    with pytest.raises(ValueError, match="expected x"):
        gated_mlp(x, wg, wu[:8], wd)
    with pytest.raises(ValueError, match="activation"):
        gated_mlp(x, wg, wu, wd, activation="swiglu")
    with pytest.raises(ValueError, match="must be on"):
        gated_mlp(x, wg.cpu(), wu, wd)
    with pytest.raises(ValueError, match="probability"):
        dropout(x, 1.0, 1)
    with pytest.raises(ValueError, match="seed"):
        dropout(x, 0.5, torch.tensor(3))
    for f, a in ((lambda t: gated_mlp(t, wg, wu, wd), x), (lambda t: layer_norm(t, wg[0]), x), (lambda t: dropout(t, 0.5, 1), x)):
        leaf = a.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(leaf).float().pow(2).sum(), [leaf], create_graph=True)
        with pytest.raises(RuntimeError):                       # no formula of second order
            torch.autograd.grad(g.float().sum(), [leaf])


def test_a_seed_that_changed_between_the_passes_is_noticed(gpu_device):
    from palimpsa_amd.ops.layer_glue import dropout, residual_layer_norm
    x, w = _randn(gpu_device, 4, 32), _randn(gpu_device, 32)
    for f in (lambda t, s: dropout(t, 0.5, s), lambda t, s: residual_layer_norm(t, None, w, dropout_p=0.5, seed=s)[0]):
        seed = torch.tensor(5, device=gpu_device)
        y = f(x.clone().requires_grad_(True), seed)
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()


# ---------------------------------------------------------------------------------------------------------- not finite
@pytest.mark.parametrize("M", [5, 300])
def test_a_row_that_is_not_finite_stays_in_its_row(gpu_device, M):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    *inp, dy = make(gpu_device, M, 64, 200, 72, BF)
    clean = [t.clone().requires_grad_(True) for t in inp]
    y0 = gated_mlp(*clean)
    (dx0,) = torch.autograd.grad(y0, clean[:1], dy)
    for bad in (float("nan"), float("inf")):
        x = inp[0].clone()
        x[M // 2, 3] = bad
        leaves = [x.requires_grad_(True)] + [t.clone().requires_grad_(True) for t in inp[1:]]
        y = gated_mlp(*leaves)
        (dx,) = torch.autograd.grad(y, leaves[:1], dy)
        rest = torch.arange(M, device=gpu_device) != M // 2
        assert not torch.isfinite(y[M // 2]).any() and torch.equal(y[rest], y0[rest]) and torch.equal(dx[rest], dx0[rest])


@pytest.mark.parametrize("M", [5, 300])
def test_a_hidden_entry_that_is_not_finite_keeps_its_neighbours_exact(gpu_device, M):
    """An infinity in one row of w_up: that hidden entry's gradients are not finite, the gradients of the seven that are kept beside it are."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    x, wg, wu, wd, dy = make(gpu_device, M, 64, 64, 64, BF)
    wu[10] = float("inf")
    wd[:, 10] = 0
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_mlp(*leaves)
    dwg, dwu = torch.autograd.grad(y, leaves[1:3], dy)
    rest = torch.arange(64, device=gpu_device) != 10
    assert torch.isfinite(dwg[rest]).all() and torch.isfinite(dwu[rest]).all()
    val, tol = fb.gated_mlp(x, wg[rest], wu[rest], wd[:, rest], "silu", BF, dy)
    # beside an infinity the others are kept in 6 bits after the leading one: errors of 2^-6 of them
    slack = 2 ** -6 * (dy.double().abs() @ wd.double().abs())[:, 8:16].abs()
    extra = torch.zeros(64, 64, dtype=torch.float64, device=gpu_device)
    g, u = (x.double() @ t.double().T for t in (wg[8:16], wu[8:16]))
    u = torch.where(torch.isfinite(u), u, 0.0)
    extra[8:16] = (slack * (1.13 + 0.8 * g.abs()) * (u.abs() + g.abs()) * 2).T @ x.double().abs()
    fb.within(dwg[rest], val["w_gate"], tol["w_gate"] + extra[rest], "dw_gate")
    fb.within(dwu[rest], val["w_up"], tol["w_up"] + extra[rest], "dw_up")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [9, 200])
def test_a_large_hidden_entry_keeps_its_neighbours_exact(gpu_device, dtype, M):
    """Hidden entries thousands of times as large as those beside them: each entry's gradients stand in proportion to itself."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    x, wg, wu, wd, dy = make(gpu_device, M, 64, 64, 64, dtype)
    wg[3] *= 300
    wu[3], wu[20], wu[21] = wu[3] * 5000, wu[20] * 2e6, wu[21] * 1e-6
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(gated_mlp(*leaves), leaves, dy)
    val, tol = fb.gated_mlp(x, wg, wu, wd, "silu", dtype, dy)
    for got, name in zip(grads, ("x", "w_gate", "w_up", "w_down")):
        fb.within(got, val[name], tol[name], name)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [9, 200])
def test_zero_factors_have_the_derivative_at_zero(gpu_device, dtype, M):
    """Weights that begin as zeros, whole and in part: relu passes no gradient at zero, silu half of it."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    x, wg, wu, wd, dy = make(gpu_device, M, 64, 96, 64, dtype)
    for rows in (slice(0, 96), slice(5, 96, 2)):
        wz = wg.clone()
        wz[rows] = 0
        for act in ("relu", "silu"):
            leaves = [t.detach().clone().requires_grad_(True) for t in (x, wz, wu, wd)]
            dx, dwg, dwu, dwd = torch.autograd.grad(gated_mlp(*leaves, act), leaves, dy)
            assert not dwu[rows].any() and not dwd[:, rows].any()
            if act == "relu":
                assert not dwg[rows].any()
                if rows == slice(0, 96):
                    assert not dx.any()
            val, tol = fb.gated_mlp(x, wz, wu, wd, act, dtype, dy)
            for got, name in zip((dx, dwg, dwu, dwd), ("x", "w_gate", "w_up", "w_down")):
                if act == "silu":          # (the bound takes relu's jump at zero for an error)
                    fb.within(got, val[name], tol[name], name)


def test_dropped_entries_are_zero_whatever_they_held(gpu_device):
    from palimpsa_amd.ops.layer_glue import dropout, residual_layer_norm
    x = _randn(gpu_device, 64, 96, dtype=BF)
    keep = fo.kept((64, 96), 0.4, 21).to(gpu_device)
    bad = torch.where(keep, x, torch.tensor(float("nan"), dtype=BF, device=gpu_device))
    bad[~keep & (torch.rand(64, 96, device=gpu_device) < 0.5)] = float("inf")
    assert torch.equal(dropout(bad, 0.4, 21), dropout(x, 0.4, 21))
    w = _randn(gpu_device, 96, seed=1)
    for a, b in zip(residual_layer_norm(bad, x, w, dropout_p=0.4, seed=21), residual_layer_norm(x, x, w, dropout_p=0.4, seed=21)):
        assert torch.equal(a, b)


def test_a_norm_of_large_and_of_equal_entries(gpu_device):
    from palimpsa_amd.ops.layer_glue import layer_norm
    w = torch.ones(768, device=gpu_device)
    x = 1e4 + _randn(gpu_device, 8, 768)                       # a mean far from zero
    val, tol = fb.layer_norm(x, w, None, 1e-5, F32)
    fb.within(layer_norm(x, w), val["y"], tol["y"], "y")
    y = layer_norm(torch.full((3, 768), 7.0, device=gpu_device, dtype=BF), w, w)
    assert torch.equal(y, torch.ones_like(y))                   # nothing but the bias
    x[2, 5] = float("nan")
    y = layer_norm(x, w)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4, 5, 6, 7]]).all()


# ------------------------------------------------------------------------------------------------- around the results
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,dim,hidden,out", [(1, 8, 24, 8), (33, 72, 136, 40), (65, 40, 72, 264), (300, 264, 200, 136)])
def test_nothing_is_written_around_the_results(gpu_device, dtype, rows, dim, hidden, out):
    """The C entry points on buffers with a margin on either side that has to stay as it was, the workspace's and the kept numbers' too."""
    from palimpsa_amd import _lib as L
    from palimpsa_amd.ops.palimpsa import _common as cm
    lib, dev, td = L.load(), gpu_device, (F32, BF)[dtype]
    guards = []

    def room(nbytes):
        t = torch.full((nbytes + 8192,), 0x5A, dtype=torch.uint8, device=dev)
        guards.append((t, nbytes))
        return C.c_void_p(t.data_ptr() + 4096)

    es = td.itemsize
    x, wg, wu, wd, dy = make(dev, rows, dim, hidden, out, td)
    d = L.PalMlpDims(rows=rows, x_stride=dim, dim=dim, hidden=hidden, out_dim=out, dtype=dtype, activation=0)
    kept = room(lib.pal_gated_mlp_kept_bytes(d))
    base = dict(x=cm._ptr(x), w_gate=cm._ptr(wg), w_up=cm._ptr(wu), w_down=cm._ptr(wd))
    s = cm.current_stream_ptr(dev)
    for keep in (0, 1):
        n = lib.pal_gated_mlp_fwd_workspace_bytes(d, keep)
        t = L.PalMlpTensors(**base, y=room(rows * out * es), kept=kept if keep else None)
        assert lib.pal_gated_mlp_fwd(d, t, room(n), n, s) == 0
    g = L.PalMlpGrads(dy=cm._ptr(dy), dx=room(rows * dim * es), dw_gate=room(hidden * dim * es), dw_up=room(hidden * dim * es), dw_down=room(out * hidden * es))
    n = lib.pal_gated_mlp_bwd_workspace_bytes(d, g)
    assert lib.pal_gated_mlp_bwd(d, L.PalMlpTensors(**base, kept=kept), g, room(n), n, s) == 0
    nd = L.PalLayerNormDims(rows=rows, x_stride=dim, res_stride=dim, dim=dim, dtype=dtype, res_dtype=0, weight_dtype=0, eps=1e-5, drop=L.PalDropout(p=0.5, seed=1))
    w = torch.ones(dim, device=dev)
    res = _randn(dev, rows, dim)
    nt = L.PalLayerNormTensors(x=cm._ptr(x), residual=cm._ptr(res), weight=cm._ptr(w), bias=cm._ptr(w), residual_out=room(rows * dim * 4), y=room(rows * dim * es),
                               stats=room(rows * 8))
    assert lib.pal_layer_norm_fwd(nd, nt, s) == 0
    n = lib.pal_layer_norm_bwd_workspace_bytes(nd)
    ng = L.PalLayerNormGrads(dy=cm._ptr(x), dresidual_out=cm._ptr(res), dx=room(rows * dim * es), dresidual=room(rows * dim * 4), dweight=room(dim * 4), dbias=room(dim * 4))
    assert lib.pal_layer_norm_bwd(nd, nt, ng, room(n), n, s) == 0
    assert lib.pal_dropout(L.PalDropout(p=0.5), cm._ptr(x), room(rows * dim * es), rows, dim, dim, dtype, s) == 0
    torch.cuda.synchronize(dev)
    for i, (t, nbytes) in enumerate(guards):
        assert (t[:4096] == 0x5A).all() and (t[4096 + nbytes:] == 0x5A).all(), i


# ---------------------------------------------------------------------------------------------------- graphs, streams
def _block(x, res, p, seed, drop=0.1):
    """Two blocks' second halves as a model calls them; p: parameters of both."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm, residual_layer_norm
    x = dropout(x, drop, seed, 0)
    for i, (w, b, wg, wu, wd) in enumerate(p):
        y, res = residual_layer_norm(x, res, w, b, dropout_p=drop, seed=seed, site=i + 1, residual_in_fp32=True)
        x = gated_mlp(y, wg, wu, wd)
    return layer_norm(x + res.to(x.dtype), p[0][0], p[0][1])


def _params(dev, D, F, dtype):
    return [[_randn(dev, D, seed=10 * i).abs() + 0.5, _randn(dev, D, seed=10 * i + 1)] +
            [(_randn(dev, *s, seed=10 * i + 2 + j) / s[1] ** 0.5).to(dtype) for j, s in enumerate(((F, D), (F, D), (D, F)))] for i in range(2)]


def test_blocks_in_full_precision(gpu_device):
    """Two blocks in fp32, forward and all gradients, against the same in 64 bits: the fp32 bar."""
    D, F, M = 96, 264, 300
    p = [[t.requires_grad_(True) for t in layer] for layer in _params(gpu_device, D, F, F32)]
    x, res, dy = (_randn(gpu_device, M, D, seed=s) for s in (50, 51, 52))
    x.requires_grad_(True)
    y = _block(x, res, p, 77)
    leaves = [x] + [t for layer in p for t in layer]
    grads = torch.autograd.grad(y, leaves, dy)

    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    wp = [wide[1:6], wide[6:11]]
    drop = lambda t, site: t * fo.kept((M, D), 0.1, 77, site).to(t.device) / 0.9  # noqa: E731
    h, r = drop(wide[0], 0), res.double()
    for i, (w, b, wg, wu, wd) in enumerate(wp):
        r = drop(h, i + 1) + r
        h = fo.gated_mlp(torch.nn.functional.layer_norm(r, (D,), w, b), wg, wu, wd)[0]
    ref = torch.nn.functional.layer_norm(h + r, (D,), wp[0][0], wp[0][1])
    assert hp.max_rel(y, ref) <= hp.FP32_REL_TOL
    for i, (g, rg) in enumerate(zip(grads, torch.autograd.grad(ref, wide, dy.double()))):
        assert hp.max_rel(g, rg) <= hp.FP32_REL_TOL, i


def test_a_captured_block_takes_a_new_seed_at_every_replay(gpu_device):
    D, F, M = 128, 256, 200
    p = _params(gpu_device, D, F, BF)
    x, res = _randn(gpu_device, M, D, seed=60, dtype=BF), _randn(gpu_device, M, D, seed=61)
    seed = torch.zeros((), dtype=torch.int64, device=gpu_device)
    side = torch.cuda.Stream()
    with torch.no_grad():
        with torch.cuda.stream(side):
            for _ in range(2):
                _block(x, res, p, seed)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _block(x, res, p, seed)
        seen = []
        for step in (3, 4, 1 << 62, 3):
            seed.fill_(step)
            x.copy_(_randn(gpu_device, M, D, seed=step % 1000, dtype=BF))
            g.replay()
            got = out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, _block(x, res, p, step)), step
            seen.append(got)
        assert torch.equal(seen[0], seen[3]) and not torch.equal(seen[0], seen[1])


@pytest.mark.parametrize("D,F,M", [(128, 256, 300), (61, 99, 70), (61, 99, 20)])
def test_a_captured_training_step(gpu_device, D, F, M):
    p = [[t.requires_grad_(True) for t in layer] for layer in _params(gpu_device, D, F, BF)]
    leaves = [t for layer in p for t in layer]
    x, res, dy = _randn(gpu_device, M, D, seed=70, dtype=BF), _randn(gpu_device, M, D, seed=71), _randn(gpu_device, M, D, seed=72, dtype=BF)
    seed = torch.zeros((), dtype=torch.int64, device=gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(_block(x, res, p, seed), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = torch.autograd.grad(_block(x, res, p, seed), leaves, dy)
    for step in (5, 6, 5):
        seed.fill_(step)
        x.copy_(_randn(gpu_device, M, D, seed=step, dtype=BF))
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = torch.autograd.grad(_block(x, res, p, step), leaves, dy)
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (step, i)
        del want


def test_two_streams_at_once(gpu_device):
    D, F, M = 256, 512, 700
    p = _params(gpu_device, D, F, BF)
    data = [(_randn(gpu_device, M, D, seed=80 + i, dtype=BF), _randn(gpu_device, M, D, seed=90 + i)) for i in range(2)]
    with torch.no_grad():
        want = [_block(x, r, p, i) for i, (x, r) in enumerate(data)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in data]
        outs = []
        for _ in range(3):
            got = []
            for i, (s, (x, r)) in enumerate(zip(streams, data)):
                with torch.cuda.stream(s):
                    got.append(_block(x, r, p, i))
            outs.append(got)
        torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------- far offsets
def test_rows_beyond_four_gigabytes(gpu_device):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm
    M, D, F = 1200000, 2048, 64                               # 4.9 GB of rows
    x = torch.zeros(M, D, dtype=BF, device=gpu_device)
    at = torch.cat([torch.arange(0, 40), torch.arange(M // 2, M // 2 + 40), torch.arange(M - 40, M)]).to(gpu_device)
    x[at] = _randn(gpu_device, 120, D, seed=1, dtype=BF)
    wg, wu, wd = ((_randn(gpu_device, *s, seed=2 + i) / s[1] ** 0.5).to(BF) for i, s in enumerate(((F, D), (F, D), (D, F))))
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_mlp(*leaves)
    dy = torch.zeros_like(y)
    dy[at] = _randn(gpu_device, 120, D, seed=9, dtype=BF)
    grads = torch.autograd.grad(y, leaves, dy)
    val, tol = fb.gated_mlp(x[at], wg, wu, wd, "silu", BF, dy[at])
    fb.within(y[at], val["y"], tol["y"], "y")
    fb.within(grads[0][at], val["x"], tol["x"], "dx")
    assert not y[60:1000].any() and not grads[0][60:1000].any()
    for n, g in zip(("w_gate", "w_up", "w_down"), grads[1:]):
        fb.within(g, val[n], tol[n], "d" + n)                  # (zero rows add nothing, not even a rounding)
    del grads, dy, y
    x = x.detach()
    with torch.no_grad():
        z = dropout(x, 0.25, 5)
        keep = fo.kept((M - (M - 40), D), 0.25, 5)             # rows are counted from the first: compare the first ones, and the last by hand
        assert torch.equal(z[:40], torch.where(keep.to(gpu_device), x[:40].float() * (1 / 0.75), 0.0).to(BF))
        share = (z[M - 40:] != 0).double().mean().item()
        assert abs(share - 0.75) < 5 * (0.75 * 0.25 / (40 * D)) ** 0.5
        w = torch.ones(D, device=gpu_device)
        val, tol = fb.layer_norm(x[at], w, None, 1e-5, BF)
        fb.within(layer_norm(x, w)[at], val["y"], tol["y"], "y")


def test_equal_calls_give_equal_bits(gpu_device):
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    *inp, dy = make(gpu_device, 2100, 192, 520, 192, BF)
    leaves = [t.requires_grad_(True) for t in inp]
    a, b = (torch.autograd.grad(gated_mlp(*leaves), leaves, dy) for _ in range(2))
    for s, t in zip(a, b):
        assert torch.equal(s, t)
