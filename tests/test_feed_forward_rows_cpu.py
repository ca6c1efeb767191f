"""The tests' dropout by explicit row numbers against the oracle's."""
import pytest
import torch

from oracle import feed_forward_oracle as fo
from tests import feed_forward_rows as fr


@pytest.mark.parametrize("rows,D", [(1, 1), (7, 5), (40, 64), (33, 771)])
@pytest.mark.parametrize("p,seed,site", [(0.1, 7, 0), (0.5, -3, 5), (0.9, 1 << 63, 0xFFFFFFFF), (0.3, 0x123456789ABCDEF0, 3)])
def test_same_places(rows, D, p, seed, site):
    want = fo.kept((rows, D), p, seed, site)
    assert torch.equal(fr.kept(torch.arange(rows), D, p, seed, site), want)
    assert torch.equal(fr.kept(torch.arange(rows // 2, rows), D, p, seed, site), want[rows // 2:])


def test_rows_beyond_32_bits_are_other_rows():
    row = torch.tensor([3, 3 + (1 << 32), 3 + (1 << 33)])
    k = fr.kept(row, 4096, 0.5, 9)
    assert torch.equal(k[:1], fo.kept((4, 4096), 0.5, 9)[3:])
    for i, j in ((0, 1), (0, 2), (1, 2)):
        assert abs((k[i] == k[j]).double().mean().item() - 0.5) < 5 * 0.5 / 64
    import numpy as np
    words = fo.philox(np.array([[2, 3, 1, 6]], dtype=np.uint64), (9, 0))[0]                    # column 8 .., row 3 + 2^32, place 6
    assert torch.equal(fr.kept(row[1:2], 12, 0.5, 9, 6)[0, 8:], torch.from_numpy(words >= np.uint64(1 << 31)))
