"""Which gradients of the gated feed-forward block are wanted, and the workspace that they take, without a GPU."""
import ctypes as C
import os

import pytest


@pytest.fixture(scope="module")
def L():
    from palimpsa_amd import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    _lib.load()
    return _lib


def test_only_gradients_of_the_projections_take_rows_of_hidden_numbers(L):
    lib, P = L.load(), C.c_void_p(0x1000)
    dims = L.PalMlpDims(rows=1 << 20, x_stride=64, dim=64, hidden=4096, out_dim=64, dtype=1, activation=0)
    rows = (1 << 20) * (4096 * 2 + 128)
    size = lambda **g: lib.pal_gated_mlp_bwd_workspace_bytes(dims, L.PalMlpGrads(dy=P, **g))  # noqa: E731
    for name in ("dx", "dw_gate", "dw_up"):
        assert size(**{name: P}) >= 2 * rows and size(**{name: P, "dw_down": P}) >= 2 * rows
    assert size(dw_down=P) < rows / 100                     # (shares of its sum over the rows at most)
    assert size() == 0
    # nothing is wanted: nothing is launched, and no workspace asked for
    t = L.PalMlpTensors(x=P, w_gate=P, w_up=P, w_down=P, kept=P)
    assert lib.pal_gated_mlp_bwd(dims, t, L.PalMlpGrads(dy=P), None, 0, None) == 0
    assert lib.pal_gated_mlp_bwd(dims, t, L.PalMlpGrads(dy=P, dx=P), None, 0, None) == L.PAL_E_WORKSPACE
