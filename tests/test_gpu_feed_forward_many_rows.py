"""Norm, dropout and copies over so many rows that every wave has several, each with numbers of its own; rows beyond 4 GB in both directions."""
import pytest
import torch

from tests import feed_forward_bounds as fb
from tests import feed_forward_rows as fr

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _make(dev, rows, D, dtype, res, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    x, dy, w, b = r(rows, D).to(dtype), r(rows, D).to(dtype), r(D), r(D)
    return x, w, b, dy, None if res is None else (2 * r(rows, D) + 0.7).to(res), None if res is None else r(rows, D).to(res)


def _check(dev, rows, D, dtype, res, p):
    from palimpsa_amd.ops.layer_glue import layer_norm, residual_layer_norm
    print(rows, D, dtype, res, p, flush=True)
    x, w, b, dy, residual, dres = _make(dev, rows, D, dtype, res, D)
    seed, site = 0x3C0FFEE + D, 7
    leaves = [t.requires_grad_(True) for t in ((x, w, b) if res is None else (x, w, b, residual))]
    if res is None:
        call = lambda: [layer_norm(x, w, b)]  # noqa: E731
    else:
        call = lambda: list(residual_layer_norm(x, residual, w, b, dropout_p=p, seed=seed, site=site))  # noqa: E731
    out = call()
    with torch.no_grad():
        for a, c in zip(call(), out):
            assert torch.equal(a, c)
    grads = torch.autograd.grad(out, leaves, [dy] if res is None else [dy, dres])
    with torch.no_grad():
        x, w, b = x.detach(), w.detach(), b.detach()
        s = x if res is None else out[1]
        if res is not None:
            xs = fr.dropped(x, p, seed, site)
            want = xs + residual.double()
            fb.within(s, want, fb.half_step(res) * want.abs() + 2 * fb.E32 * (xs.abs() + residual.double().abs()), "s")
        val, tol = fb.layer_norm(s, w, b, 1e-5, dtype, dy, dres)
        fb.within(out[0], val["y"], tol["y"], "y")
        if res is not None:
            fb.within(grads[3], val["ds"], tol["ds"] + fb.half_step(res) * val["ds"].abs(), "dresidual")
        dx, edx = fr.dropped(val["ds"], p, seed, site), fr.dropped(tol["ds"], p, seed, site)
        fb.within(grads[0], dx, edx + (fb.half_step(dtype) + 2 * fb.E32) * dx.abs(), "dx")
        # The sums over the rows by the additions that a term passes through, not by as many as there are rows: a row that is left out or counted twice shows.
        from oracle import feed_forward_oracle as fo
        hat = fo.layer_norm(s, w, b)[1]
        loose = (rows + 8) * fb.E32 * (dy.double() * hat).abs().sum(0)
        n = fr.depth(rows, D) * fb.E32
        fb.within(grads[1], val["weight"], tol["weight"] - loose + n * (dy.double() * hat).abs().sum(0), "dweight")
        fb.within(grads[2], val["bias"], n * dy.double().abs().sum(0), "dbias")


# three rows a wave in the forward (8192 waves) and in the backward (4096 to 1024)
@pytest.mark.parametrize("D", [7, 64, 500, 768, 1531, 1536, 2048])
@pytest.mark.parametrize("dtype,res,p", [(BF, None, 0.0), (F32, None, 0.0), (BF, F32, 0.0), (BF, F32, 0.3), (BF, BF, 0.3), (F32, F32, 0.3)])
def test_waves_with_several_rows(gpu_device, D, dtype, res, p):
    _check(gpu_device, 24700, D, dtype, res, p)


# a workgroup a row: 2048 in the forward, 512 or 256 in the backward
@pytest.mark.parametrize("D", [2049, 2056, 4096, 4100, 8192, 8200, 16384])
@pytest.mark.parametrize("dtype,res,p", [(BF, None, 0.0), (F32, None, 0.0), (BF, F32, 0.0), (BF, F32, 0.3), (BF, BF, 0.3), (F32, F32, 0.3)])
def test_workgroups_with_several_rows(gpu_device, D, dtype, res, p):
    _check(gpu_device, 6200, D, dtype, res, p)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_copies_of_many_rows(gpu_device, dtype):
    """Workgroups of the copying kernel with several rows: 2048 of four rows of more than 504 entries, of 32 of 64."""
    import ctypes as C

    from palimpsa_amd import _lib as L
    sizes = [(20011, 515, 20016, 520), (70001, 61, 70008, 64), (20011, 1030, 20011, 1030)]
    src = [torch.randn(r, c, device=gpu_device).to(dtype) for r, c, _, _ in sizes]
    dst = [torch.full((r8, c8), 7.0, dtype=dtype, device=gpu_device) for _, _, r8, c8 in sizes]
    m = (L.PalMatrixCopy * 3)(*[L.PalMatrixCopy(src=s.data_ptr(), dst=d.data_ptr(), src_ld=c, dst_ld=c8, rows=r, cols=c, dst_rows=r8, dst_cols=c8)
                                for s, d, (r, c, r8, c8) in zip(src, dst, sizes)])
    assert L.load().pal_copy_matrices(m, 3, int(dtype == BF), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    for s, d, (r, c, _, _) in zip(src, dst, sizes):
        assert torch.equal(d[:r, :c], s) and not d[r:].any() and not d[:, c:].any()


# ---------------------------------------------------------------------------------------------------- rows beyond 4 GB
M, D = 1200000, 2048                              # 4.9 GB of bf16 rows, 9.8 of fp32


def _rows(dev):
    return torch.cat([torch.arange(0, 40), torch.arange(M // 2, M // 2 + 40), torch.arange(M - 40, M)]).to(dev)


def _filled(dev, at, seed, dtype):
    t = torch.zeros(M, D, dtype=dtype, device=dev)
    t[at] = torch.randn(at.numel(), D, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)
    return t


def test_dropout_of_far_rows(gpu_device):
    from palimpsa_amd.ops.layer_glue import dropout
    at, p, seed, site = _rows(gpu_device), 0.25, 5 << 40, 9
    x, dy = _filled(gpu_device, at, 1, BF), _filled(gpu_device, at, 2, BF)
    keep = fr.kept(at, D, p, seed, site)
    x.requires_grad_(True)
    y = dropout(x, p, seed, site)
    (dx,) = torch.autograd.grad(y, [x], dy)
    with torch.no_grad():
        for got, src in ((y, x), (dx, dy)):
            assert torch.equal(got[at], torch.where(keep, src[at].float() * (1 / (1 - p)), 0.0).to(BF))
            assert not got[1000:100000].any()


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_norm_of_a_far_stream(gpu_device, p):
    from palimpsa_amd.ops.layer_glue import residual_layer_norm
    at, seed, site = _rows(gpu_device), 5 << 40, 9
    x, dy = (_filled(gpu_device, at, i, BF).requires_grad_(i == 1) for i in (1, 2))
    res, dres = (_filled(gpu_device, at, i, F32).requires_grad_(i == 3) for i in (3, 4))
    w = torch.randn(D, generator=torch.Generator().manual_seed(6)).to(gpu_device).requires_grad_(True)
    y, s = residual_layer_norm(x, res, w, None, dropout_p=p, seed=seed, site=site)
    gx, gr, gw = torch.autograd.grad([y, s], [x, res, w], [dy, dres])
    with torch.no_grad():
        drop = (lambda t: torch.where(fr.kept(at, D, p, seed, site), t.double() * (1 / (1 - p)), 0.0)) if p else (lambda t: t.double())
        want = drop(x[at]) + res[at].double()
        fb.within(s[at], want, 3 * fb.E32 * (drop(x[at]).abs() + res[at].double().abs()), "s")
        val, tol = fb.layer_norm(s[at], w, None, 1e-5, BF, dy[at], dres[at])
        fb.within(y[at], val["y"], tol["y"], "y")
        fb.within(gr[at], val["ds"], tol["ds"] + fb.E32 * val["ds"].abs(), "dresidual")
        dx = drop(val["ds"])
        fb.within(gx[at], dx, drop(tol["ds"]) + (2 ** -8 + 2 * fb.E32) * dx.abs(), "dx")
        fb.within(gw, val["weight"], tol["weight"], "dweight")           # (rows of zeros add nothing, not even a rounding)
        for t in (y, s, gr, gx):
            assert not t[1000:100000].any()


def test_norm_of_far_rows(gpu_device):
    from palimpsa_amd.ops.layer_glue import layer_norm
    at = _rows(gpu_device)
    x, dy = (_filled(gpu_device, at, i, BF).requires_grad_(i == 1) for i in (1, 2))
    w, b = (torch.randn(D, generator=torch.Generator().manual_seed(i)).to(gpu_device).requires_grad_(True) for i in (6, 7))
    y = layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], dy)
    with torch.no_grad():
        val, tol = fb.layer_norm(x[at], w, b, 1e-5, BF, dy[at])
        fb.within(y[at], val["y"], tol["y"], "y")
        fb.within(gx[at], val["ds"], tol["ds"] + 2 ** -8 * val["ds"].abs(), "dx")
        fb.within(gw, val["weight"], tol["weight"], "dweight")
        fb.within(gb, val["bias"], tol["bias"], "dbias")
        assert torch.equal(y[1000:2000], b.detach().to(BF).expand(1000, D)) and not gx[1000:100000].any()
