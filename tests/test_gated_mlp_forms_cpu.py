"""Which tile forms the sizes of the GPU tests take: every one that the plan gives to a product, so that a change of its constants cannot take one out of the
tests unseen."""
import os

import pytest

from tests import gated_mlp_forms as gf


@pytest.fixture(scope="module")
def L():
    from palimpsa_amd import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    _lib.load()
    return _lib


def _all(dtype):
    """Every product by every form, k whole and in shares, one tile a workgroup and several; without what only sizes beyond 10^11 operations take."""
    wide = {(256, 256), (256, 192), (128, 128)} | ({(64, 64)} if dtype == "fp32" else set())
    gated = {(256, 128), (128, 64)} | ({(64, 64)} if dtype == "fp32" else set())
    keys = {(p, *t, s, r) for p in gf.PRODUCTS for t in (gated if p == "up" else wide) for s in (False, True) for r in (False, True)}
    if dtype == "bf16":
        keys -= {("up", 256, 128, True, True), ("down", 256, 192, True, True), ("down", 256, 256, True, True), ("grad", 256, 192, True, True),
                 ("grad", 256, 256, True, False), ("grad", 256, 256, True, True)}
    return keys


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_every_form_is_taken(L, dtype):
    seen = set().union(*(gf.taken(L, *s, dtype) for s in gf.SIZES[dtype]))
    assert _all(dtype) <= seen, sorted(_all(dtype) - seen)


def test_the_kernels_of_few_rows_are_taken(L):
    assert all("up" not in gf.forms(L, *s, dtype) and "grad" in gf.forms(L, *s, dtype) for s in gf.FEW for dtype in ("bf16", "fp32") if s[0] <= 17)
    assert any(s[0] > 48 and "up" not in gf.forms(L, *s, "bf16") for s in gf.FEW)


def test_forms_refuse(L):
    lib, f = L.load(), L.PalMlpForms()
    d = L.PalMlpDims(rows=64, x_stride=64, dim=64, hidden=128, out_dim=64, dtype=1, activation=0)
    assert lib.pal_gated_mlp_forms(None, None, f) == L.PAL_E_NULL and lib.pal_gated_mlp_forms(d, None, None) == L.PAL_E_NULL
    d.dim = 5
    assert lib.pal_gated_mlp_forms(d, None, f) == L.PAL_E_DIM
    d.dim, d.rows = 64, 200
    assert lib.pal_gated_mlp_forms(d, None, f) == 0 and f.tile_rows[0] and f.tile_rows[1] and not any(f.tile_rows[2:])
