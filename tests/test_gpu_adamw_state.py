"""GPU tests of what AdamW keeps between steps: its counters and moments when a step is
refused, saved and loaded state, version counters, tensors named twice."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_versions_of_all_that_is_written(fms):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    c = p.bfloat16()
    m, v = fms.moments8(p), fms.moments8(p)
    written = [p, c, *m, *v]
    before = [t._version for t in written]
    fms.adamw_step([p], [g], [m], [v], step=1, copies=[c])
    assert all(t._version > b for t, b in zip(written, before))
    assert g._version == 0
