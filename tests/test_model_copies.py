"""Copies of a model (copy.deepcopy, torch.save of the module) and the tags of their forward calls."""
import copy
import pickle

import pytest
import torch

from dgcnn_amd.model import Model


@pytest.mark.parametrize("make", [copy.deepcopy, lambda m: pickle.loads(pickle.dumps(m)), copy.copy])
def test_a_copys_forward_tags_do_not_meet_the_originals(make):
    """an error word that the original's batch left in memory must not read as one of the copy's"""
    m = Model(3, 2)
    for _ in range(5):
        m._next_epoch()
    copies = [make(m) for _ in range(8)]
    starts = [m._epoch] + [c._epoch for c in copies]
    gaps = [abs(a - b) for i, a in enumerate(starts) for b in starts[:i]]
    assert min(min(g, 0x7FFFFFFE - g) for g in gaps) > 1 << 20
    for c in copies:
        assert 0 < c._next_epoch() <= 0x7FFFFFFE
        assert all(torch.equal(p, q) for p, q in zip(m.state_dict().values(), c.state_dict().values()))


def test_a_copy_does_not_look_for_the_originals_errors():
    """the workspace that a copy took along is the original's business: its tags are not the copy's"""
    m = Model(3, 2)
    m.__dict__["_last_ws"], m.__dict__["_last_dims"] = torch.zeros(16, dtype=torch.uint8), (1, 0, 1, 3, 2)
    c = copy.deepcopy(m)
    assert c._last_ws is None and c._last_dims is None and m._last_ws is not None
    c.check_errors()
