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


# rows x columns of every form that the preference loss has: one pass per pair and gradient, rows in one workgroup or in one run;
# pairs of their own kernel, rows in one workgroup or in several runs
PAIR_FORMS = [(30, 50), (30, 8192), (30, 40001), (1300, 50), (300, 40001)]


def pair_inputs(rows, cols, seed, pairs=4):
    r, z, t = make(rows, cols, seed)
    cuts = np.linspace(0, rows, 2 * pairs + 1).astype(int)
    cuts[1:-1] += r.integers(0, 2, 2 * pairs - 1)                 # ragged, two tokens at least
    refl = (target_logp(z, t) + 0.3 * r.standard_normal(rows)).astype(np.float32)
    return z, t, cuts, refl


@pytest.mark.parametrize("rows,cols", PAIR_FORMS)
@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
def test_sigmoid_loss_of_an_infinite_gap(ops, rows, cols, eps):
    """An answer with a token that cannot be chosen has the score -inf.  -log sigmoid(inf) is 0, and a term whose factor is 0 is
    not there: the loss is 0 where the preferred side wins for certain, infinite where it loses."""
    z, t, starts, refl = pair_inputs(rows, cols, cols + 41)
    for side in (3, 4):                                           # pair 1: its rejected answer; pair 2: its chosen one
        row = starts[side]
        z[row, t[row]] = -np.inf
    got = ops.preference_grad(dev(z), dev(t), dev(starts.astype(np.uint32)), ref_logp=dev(refl), beta=0.3, label_smoothing=eps)
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol = ref.preference(z, t, starts, ref=refl, beta=0.3, eps=eps)
    want["loss"][1] = 0.0 if eps == 0 else np.inf
    want["loss"][2] = 0.0 if eps == 1 else np.inf
    assert want["scores"][3] == -np.inf and want["scores"][4] == -np.inf and np.isfinite(want["grad"]).all()
    tol["loss"][1:3] = 0.0
    compare(dict(grad=got[0], loss=got[1], scores=got[2]), (want, tol), f"{rows} x {cols}")


@pytest.mark.parametrize("rows,cols", PAIR_FORMS)
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
def test_a_pair_without_a_score_shows_it(ops, rows, cols, kind):
    """NaN in one entry of ref_logp: the loss of its pair and the gradients of all of the pair's supervised rows are NaN, which a
    step's checks see; the other pairs keep their bits."""
    z, t, starts, refl = pair_inputs(rows, cols, cols + 43)
    t[starts[2] + 1] = cols                                       # one row of the pair that is not supervised, beside the last ones
    live = ref.supervised(rows, cols, t, None, starts)
    spoilt = refl.copy()
    spoilt[starts[3]] = np.nan                                    # (a rejected answer; its pair is rows starts[2] to starts[4])

    def run(refl):
        got = ops.preference_grad(dev(z), dev(t), dev(starts.astype(np.uint32)), ref_logp=dev(refl), kind=kind, beta=0.3)
        return [a.cpu().numpy() for a in got]
    (g0, l0, s0), (g, l, s) = run(refl), run(spoilt)
    pair = np.zeros(rows, bool)
    pair[starts[2]:starts[4]] = True
    assert live[starts[3]] and np.isfinite(g0).all() and np.isfinite(l0).all() and np.isfinite(s0).all()
    assert np.isnan(g[pair & live]).all() and (g[pair & ~live] == 0).all() and np.array_equal(g[~pair], g0[~pair])
    assert np.array_equal(np.isnan(l), np.arange(4) == 1) and np.array_equal(l[[0, 2, 3]], l0[[0, 2, 3]])
    assert np.array_equal(np.isnan(s), np.arange(8) == 3) and np.array_equal(np.delete(s, 3), np.delete(s0, 3))


@pytest.mark.parametrize("rows,cols", [(7, 13), (5, 33001)])
def test_buffers_that_touch(ops, rows, cols):
    """Slices of one allocation, each starting where the one before ends, share nothing."""
    r, z, t = make(rows, cols, cols + 47)
    adv, old, refl = policy_inputs(r, z, t)
    w = (0.5 + r.random(rows)).astype(np.float32)
    parts = [adv, np.full(z.shape, np.nan, np.float32), old, z, refl, w]
    room = torch.empty(sum(p.size for p in parts), device="cuda")
    views, at = [], 0
    for p in parts:
        views.append(room[at:at + p.size].view(p.shape))
        views[-1].copy_(torch.from_numpy(p))
        at += p.size
    a, grad, o, Z, R, W = views
    got = ops.policy_grad(Z, dev(t), a, o, rows, ref_logp=R, weights=W, clip=(0.2, 0.3), kl_coef=0.05, grad=grad)
    want = ref.policy(z, t, adv, old, rows, ref=refl, weights=w, clip=(0.2, 0.3), kl_coef=0.05)
    compare(dict(zip(("grad", "loss", "logp", "kl"), got)), want, f"{cols}")
    for view, p in zip((a, o, Z, R, W), (adv, old, z, refl, w)):
        assert np.array_equal(view.cpu().numpy(), p)


def test_kl_estimate_far_from_the_reference(ops):
    """k(d) = e^d - 1 - d over the range of FP32.  In rows of one column logp is 0 up to the 1e-7 of a row's logarithm, so d is ref_logp up
    to that, which changes k by at most 1e-7 |e^d - 1|.  Beyond |d| = 1 an exponential good to a step of its last place (2^-23, and half
    of that for rounding its argument's fraction) and the difference's rounding remain; below, the terms of the series: six
    half steps for their products and sums, one for what is cut off, one for the last product."""
    d = np.concatenate([np.linspace(-100.0, 88.0, 1501), np.linspace(-1.5, 1.5, 401), np.geomspace(1e-3, 1.0, 60), -np.geomspace(1e-3, 1.0, 60)]).astype(np.float32)
    rows = len(d)
    z, t, zero = np.linspace(-3, 3, rows).astype(np.float32)[:, None], np.zeros(rows, np.uint32), np.zeros(rows, np.float32)
    _, loss, logp, kl, _ = ops.policy_grad(dev(z), dev(t), dev(zero), dev(zero), rows, ref_logp=dev(d), kl_coef=0.5)
    d = d.astype(np.float64)
    rise = np.expm1(d)
    # e^d - 1 - d without its cancellation
    want = np.where(np.abs(d) < 1e-2, d * d * (0.5 + d * (1 / 6 + d * (1 / 24 + d * (1 / 120 + d / 720)))), rise - d)
    far = np.abs(d) >= 1
    tol = 1e-7 * np.abs(rise) + 1e-14 * np.exp(d) + ref.HALF_STEP * np.where(far, 3 * np.exp(d) + 2 * want, 8 * want)
    assert np.abs(logp.cpu().numpy()).max() <= 1e-7
    check("k", kl, want, tol)
    check("loss", loss, 0.5 * want, 0.5 * tol + ref.HALF_STEP * 0.5 * want)


@pytest.mark.parametrize("rows,cols", PAIR_FORMS + [(520, 151936)])
def test_preference_over_the_logits_and_its_log_probabilities(ops, rows, cols):
    """The gradient written over the logits, as a training step has it, and the optional log-probabilities, in every form; rows ahead of
    the first sequence, behind the last and in between that are not supervised have 0."""
    z, t, starts, refl = pair_inputs(rows, cols, cols + 53)
    starts = starts.copy()
    starts[0], starts[-1] = 1, rows - 1
    t[starts[2] + 1] = cols
    live = ref.supervised(rows, cols, t, None, starts)
    kw = dict(ref_logp=dev(refl), beta=0.3, label_smoothing=0.1, average=True)
    S, T = dev(starts.astype(np.uint32)), dev(t)
    plain = ops.preference_grad(dev(z), T, S, **kw)
    Z, logp = dev(z), torch.full((rows,), float("nan"), device="cuda")
    inside = ops.preference_grad(Z, T, S, grad=Z, logp=logp, **kw)
    assert inside[0] is Z and all(torch.equal(a, b) for a, b in zip(plain, inside))
    want, tol = ref.token_logprobs(z, np.where(live, t, np.uint32(cols)))
    check("logp", logp, want["logp"], tol["logp"])
    if rows * cols < 2e7:
        compare(dict(zip(("grad", "loss", "scores"), inside)), ref.preference(z, t, starts, ref=refl, beta=0.3, eps=0.1, average=True), f"{rows} x {cols}")


def test_refused_log_probabilities(ops):
    from seraph_amd._lib import SeraphError
    z, t, s = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    f = torch.zeros(4, device="cuda")
    for bad in (f[:3], f.double(), f.cpu(), f.expand(2, 4)[:, 0], z[:, 0]):
        with pytest.raises(SeraphError, match="logp"):
            ops.preference_grad(z, t, s, logp=bad)
    for bad in (dict(logp=f, ref_logp=f), dict(logp=z.view(-1)[4:8])):
        with pytest.raises(SeraphError, match="overlap"):
            ops.preference_grad(z, t, s, **bad)
