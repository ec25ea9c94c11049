"""Arguments of the trainer's objective steps that are missing or do not fit are refused with the package's error, before any call."""
import numpy as np
import pytest


@pytest.fixture()
def t():
    from seraph_amd.trainer import Trainer
    bare = Trainer.__new__(Trainer)                               # no device, no handle: whatever reaches the library is refused there
    bare._h = None
    return bare


def test_a_teacher_without_a_list(t):
    from seraph_amd._lib import SeraphError
    tok, starts, ids, z = np.zeros(6, np.int32), np.array([0, 3, 6], np.int32), np.zeros((6, 2), np.uint32), np.zeros((6, 2), np.float32)
    for a, b in ((None, z), (ids, None), (None, None), (ids[:, :1], z), (ids[:5], z), (ids, z[:, 0]), (ids[:, 0], z)):
        with pytest.raises(SeraphError, match="teacher"):
            t.step_distill(tok, starts, a, b)
    with pytest.raises(SeraphError, match="teacher_lse"):
        t.step_distill(tok, starts, ids, z, teacher_lse=z)
