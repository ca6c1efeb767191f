"""Padding of the hidden dim in the C entry points of the gated feed-forward block, without a GPU."""
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


def test_padding_is_less_than_eight_columns(L):
    lib, P = L.load(), C.c_void_p(0x1000)
    dims = lambda pad: L.PalMlpDims(rows=64, x_stride=64, dim=64, hidden=128, out_dim=64, dtype=1, activation=0, hidden_pad=pad)  # noqa: E731
    t = L.PalMlpTensors(x=P, w_gate=P, w_up=P, w_down=P, y=P, kept=P)
    g = L.PalMlpGrads(dy=P, dx=P)
    for pad in (-1, 8, 128):
        assert lib.pal_gated_mlp_kept_bytes(dims(pad)) == 0
        assert lib.pal_gated_mlp_fwd(dims(pad), t, P, 1 << 40, None) == L.PAL_E_DIM
        assert lib.pal_gated_mlp_bwd(dims(pad), t, g, P, 1 << 40, None) == L.PAL_E_DIM
    sizes = {pad: (lib.pal_gated_mlp_kept_bytes(dims(pad)), lib.pal_gated_mlp_fwd_workspace_bytes(dims(pad), 0), lib.pal_gated_mlp_bwd_workspace_bytes(dims(pad), g))
             for pad in range(8)}
    assert len(set(sizes.values())) == 1 and all(sizes[0])
