"""What a backward pass asks of the tensors that it saved, without a GPU."""
import pytest
import torch

from palimpsa_amd.ops.palimpsa import _common as cm


def test_saved_tensors_have_to_come_back_as_large_as_they_were():
    x, w = torch.zeros(6, 8), torch.zeros(8, dtype=torch.bfloat16)
    form = cm.saved_form(x, w, None)
    cm.check_saved((x, w, None), form, "op")
    cm.check_saved((torch.zeros(6, 16)[:, :8], w.clone(), None), form, "op")          # wherever they lie
    for bad in ((torch.cat([x, x]), w, None), (x[:3], w, None), (x.reshape(8, 6), w, None), (x, w.float(), None), (x, w.repeat(2), None), (x, w, w),
                (None, w, None), (x.to("meta"), w, None)):
        with pytest.raises(ValueError, match="op backward: a saved tensor came back"):
            cm.check_saved(bad, form, "op")
