"""Tables of packed batches that a captured graph reads: kept as long as their cu_seqlens tensor, whatever other batches come along."""
import gc
import weakref

import pytest
import torch

from palimpsa_amd.ops.palimpsa import _common as cm

CPU = torch.device("cpu")


def others():
    """Twenty more batches, all of them alive."""
    cus = [torch.tensor([0, 10 + i, 100]) for i in range(20)]
    for cu in cus:
        cm.chunk_meta(cu, 100, CPU)
    return cus


@pytest.mark.parametrize("forget", [others, cm.invalidate_chunk_meta, lambda: (cm.invalidate_chunk_meta(), others())])
def test_a_captured_table_is_not_freed(monkeypatch, forget):
    cu = torch.tensor([0, 40, 100])
    cm.chunk_meta(cu, 100, CPU)                    # the eager call in front of the capture
    monkeypatch.setattr(cm, "_capturing", lambda device: True)
    table = cm.chunk_meta(cu, 100, CPU)[0][3:]     # what a graph reads: a view of the memory
    memory = weakref.ref(table._base)
    want = table.clone()
    del table
    monkeypatch.setattr(cm, "_capturing", lambda device: False)
    forget()
    gc.collect()
    assert memory() is not None and torch.equal(memory()[3:], want)
    del cu
    gc.collect()
    cm.invalidate_chunk_meta()
    assert memory() is None and not cm._captured_meta


def test_captures_of_one_tensor_share_its_table(monkeypatch):
    cu = torch.tensor([0, 40, 100])
    monkeypatch.setattr(cm, "_capturing", lambda device: True)
    assert cm.chunk_meta(cu, 100, CPU)[0] is cm.chunk_meta(cu, 100, CPU)[0]
    assert [len(v[1]) for v in cm._captured_meta.values()] == [1]


def test_nothing_is_kept_outside_a_capture():
    cu = torch.tensor([0, 40, 100])
    memory = weakref.ref(cm.chunk_meta(cu, 100, CPU)[0])
    alive = others()
    gc.collect()
    assert len(alive) == 20 and memory() is None and id(cu) not in cm._captured_meta
