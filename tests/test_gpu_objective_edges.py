"""The objectives over logits at the edges of their values: reference log-probabilities of masked tokens, gaps that are
infinite or not a number.  Expected values come from the definitions, tolerances from tests/objectives_ref.py."""
import numpy as np
import pytest
import torch

from tests import objectives_ref as ref
from tests.test_gpu_objectives import check, compare, dev, make, ops, policy_inputs, run_policy, target_logp      # noqa: F401

pytestmark = pytest.mark.gpu

LOWEST = float(np.finfo(np.float32).min)


@pytest.mark.parametrize("cols", [9, 8192, 33001, 1300003])
@pytest.mark.parametrize("ent", [0.0, 0.01])
def test_kl_term_of_tokens_that_the_reference_masks(ops, cols, ent):
    """d = ref_logp - logp far below zero: the slope of the KL term is e^d - 1 = -1, also where k itself is infinite."""
    masks = np.array([-20.0, -1e4, -3e7, -1e9, LOWEST, -np.inf], np.float32)
    rows = len(masks) if cols < 10 ** 6 else 3
    r, z, t = make(rows, cols, cols + 31)
    adv, old, _ = policy_inputs(r, z, t)
    refl = masks[-rows:].copy()
    adv[rows // 2] = 0.0                                          # the KL term alone
    got = run_policy(ops, z, t, adv, old, rows, refl=refl, kl=0.25, ent=ent)
    with np.errstate(over="ignore"):
        want = ref.policy(z, t, adv, old, rows, ref=refl, clip=(0.2, 0.3), kl_coef=0.25, entropy_coef=ent)
    assert np.isfinite(want[0]["grad"]).all()
    compare(got, want, f"{cols}")
