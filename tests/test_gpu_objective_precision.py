"""What the objectives over logits owe to the digits they carry: scores whose errors add up over tokens, log-probabilities within a
bound that counts the lanes a row really has, and gradients against differences that see every term."""
import numpy as np
import pytest
import torch

from tests import objectives_ref as ref
from tests.test_gpu_objectives import check, dev, distill_inputs, make, ops, policy_inputs, run_distill, run_policy, target_logp      # noqa: F401

pytestmark = pytest.mark.gpu

# log2(e) rounded to FP32 is off by this much of itself.  An exponential of d = z - m formed with it is off by d times that, always the same
# way, and the logarithm of a sum of them by the mean of m - z under the softmax times that.
ONE_PART = abs(float(np.float32(np.log2(np.e))) / np.log2(np.e) - 1.0)


@pytest.mark.parametrize("rows,cols", [(1024, 8192), (256, 40001), (1024, 40001)])
def test_errors_of_scores_do_not_add_up(ops, rows, cols):
    """Scores of one token each are the errors of log-probabilities, undisturbed by the output's rounding: the reference is the exact value,
    rounded.  Rows with a third of their mass on the largest logit and the rest far below show a bias of the exponentials best: with
    log2(e) in one float it would be about 7e-8 a token.  The bar is half of that; the mean of n random errors (some 1e-7 each:
    a few half steps of 6e-8 where a row's parts are added) lies within a third of it.  Where the row is held by one workgroup their
    spread is bounded too: a log-probability in FP32, between 8 and 16, would be off by 2^-20 / sqrt(12) = 2.8e-7."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    z = torch.empty(rows, cols, device="cuda").normal_(generator=g)
    t = torch.randint(1, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
    z[:, 0] = float(np.log(cols))
    exact = torch.log_softmax(z.double(), 1)
    want = exact.gather(1, t.long()[:, None])[:, 0]
    bias = float((exact.exp() * (z.amax(1, keepdim=True) - z).double()).sum(1).mean()) * ONE_PART
    assert bias > 6e-8
    reference = want.float()
    starts = torch.arange(0, rows + 2, 2, dtype=torch.int32, device="cuda")
    _, _, scores = ops.preference_grad(z, t, starts, ref_logp=reference)
    err = scores.double() - (want - reference.double())[0::2]
    assert abs(float(err.mean())) <= bias / 2
    if cols <= 32768:
        assert float(err.square().mean().sqrt()) <= 1.5e-7
    # the same rows as two long answers
    starts = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
    _, _, scores = ops.preference_grad(z, t, starts, ref_logp=reference)
    diff = want - reference.double()
    for q, (a, b) in enumerate(((0, rows // 2), (rows // 2, rows))):
        assert abs(float(scores[q].double() - diff[a:b - 1].sum())) <= (b - 1 - a) * bias / 2


def row_lanes(rows, cols):
    """Lanes among which token_logprobs shares a row: a workgroup's, or those of all of its runs."""
    if cols <= 32768:
        return 256 if cols <= 12 * 1024 + 3 else 512
    if rows <= 256 and cols <= 163840:
        return 1024
    return 256 * min(64, max(1, min(-(-8192 // rows), cols // 4 // 2048)))


@pytest.mark.parametrize("rows,cols", [(40, 13), (40, 1000), (40, 8192), (40, 12289), (40, 32768), (40, 50021), (300, 50021), (8, 151936), (300, 151936), (2, 1300003)])
def test_log_probabilities_within_what_their_lanes_allow(ops, rows, cols):
    """An error of e_j counts with its share p_j of the sum: with u = 2^-24, 2u (m - z_j) for the rounded difference and the rounded product,
    2u for the exponential.  Every lane adds its values one after another, each addition u of the lane's sum at most, then come 6
    additions over a wave, 8 or 16 over a workgroup, 6 and a rescaling (4) over runs or a lane's batches; the result is rounded once."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
    exact = torch.log_softmax(z.double(), 1)
    want = exact.gather(1, t.long()[:, None])[:, 0]
    below = (exact.exp() * (z.amax(1, keepdim=True) - z).double()).sum(1)
    per_lane = -(-cols // row_lanes(rows, cols)) + 4              # a head or tail value and an unfinished vector
    rescaled = 0 if cols <= 32768 else 4 * -(-per_lane // 32)     # a lane's running sum meets a new maximum at most once in 32 values
    u = ref.HALF_STEP * (2 * below + 2 + per_lane + 6 + 16 + 10 + rescaled)
    got, _, _ = ops.token_logprobs(z, t)
    assert ((got.double() - want).abs() <= u + ref.HALF_STEP * want.abs()).all()


@pytest.mark.parametrize("cols", [13, 8192, 40001])
def test_gradients_against_extrapolated_differences(ops, cols):
    """(4 D(h/2) - D(h)) / 3 of each op's own loss, D the central difference, at three columns that all hold a good share of the row.  What the
    formula itself is off by is formed in 64 bits from the definition at the same points; a loss that is off by l moves it by
    3 l / h.  The KL and entropy terms of the policy loss, the soft and the hard part of the distillation are each larger than
    four times the bar, so that none of them can be missing or wrong by a quarter."""
    rows, h = 2, 0.25
    r, z, t = make(rows, cols, cols + 61, spread=0.5)
    others = np.stack([r.choice(np.setdiff1d(np.arange(cols), [t[i]]), 2, replace=False) for i in range(rows)])
    probes = np.concatenate([t[:, None].astype(int), others], 1)
    for i in range(rows):
        z[i, probes[i]] = np.log(cols) + np.array([0.0, 0.3, -0.3])
    z = (np.round(z * 64) / 64).astype(np.float32)                # steps of h are exact
    adv, _, _ = policy_inputs(r, z, t)
    logp = target_logp(z, t)
    old, refl = logp.astype(np.float32), (logp + np.array([0.5, -0.6])).astype(np.float32)
    starts = np.array([0, 2, 4], np.uint32)
    ids = probes.astype(np.uint32)
    teacher = torch.from_numpy(np.array([[1.0, -1.0, 0.5], [-0.5, 1.5, 0.0]], np.float32))
    z4, t4, r4 = np.repeat(z, 2, 0), np.repeat(t, 2), np.repeat(refl, 2)      # a supervised and a last row for each side

    def policy(x, kl=0.5, ent=0.3):
        got = run_policy(ops, x, t, adv, old, 1, refl=refl, kl=kl, ent=ent)
        return got["loss"].cpu().numpy().astype(np.float64), got["grad"].cpu().numpy().astype(np.float64)

    def policy64(x, kl=0.5, ent=0.3):
        return ref.policy(x, t, adv, old, 1, ref=refl, clip=(0.2, 0.3), kl_coef=kl, entropy_coef=ent)

    def pref(x):
        z4[0::2] = x
        g, loss, _ = ops.preference_grad(dev(z4), dev(t4), dev(starts), ref_logp=dev(r4), beta=2.0)
        return np.repeat(loss.cpu().numpy().astype(np.float64), rows), g.cpu().numpy().astype(np.float64)[0::2]

    def pref64(x):
        w = z4.astype(np.float64)
        w[0::2] = x
        out, tol = ref.preference(w, t4, starts.astype(int), ref=r4, beta=2.0)
        return [dict(loss=np.repeat(a["loss"], rows), grad=a["grad"][0::2]) for a in (out, tol)]

    def dist(x, soft=1.0, hard=0.4):
        got = run_distill(ops, x, ids, teacher, 1, temperature=1.5, soft_coef=soft, hard_coef=hard, targets=t)
        return got["loss"].cpu().numpy().astype(np.float64), got["grad"].cpu().numpy().astype(np.float64)

    def dist64(x, soft=1.0, hard=0.4):
        return ref.distill(x, ids, teacher.numpy(), 1, temperature=1.5, soft=soft, hard=hard, targets=t)

    def extrapolated(loss, row, c):
        def at(step):
            x = z.copy()
            x[row, c] += step
            return loss(x)[row]
        wide, narrow = (at(h) - at(-h)) / (2 * h), (at(h / 2) - at(-h / 2)) / h
        return (4 * narrow - wide) / 3

    for f, f64, without in ((policy, policy64, (dict(kl=0.0), dict(ent=0.0))), (pref, pref64, ()), (dist, dist64, (dict(soft=0.0), dict(hard=0.0)))):
        out, tol = f64(z)
        _, grad = f(z)
        worst = 0.0
        for row in range(rows):
            for c in probes[row]:
                formula = extrapolated(lambda x: f64(x)[0]["loss"], row, c) - out["grad"][row, c]
                bar = abs(formula) + 3 * tol["loss"][row] / h + tol["grad"][row, c]
                got = extrapolated(lambda x: f(x)[0], row, c)
                assert abs(got - grad[row, c]) <= bar, (f.__name__, row, c, got, grad[row, c], bar)
                worst = max(worst, bar)
        for kw in without:                                        # the bar sees each term
            less = f64(z, **kw)[0]["grad"]
            assert np.abs(out["grad"] - less)[np.arange(rows)[:, None], probes].max() > 4 * worst, (f.__name__, kw, worst)


@pytest.mark.parametrize("rows,cols,calls", [(256, 151936, 8), (300, 151936, 8), (2048, 8192, 2), (2048, 40001, 2)])
def test_a_row_takes_one_exponential_for_each_logit(ops, rows, cols, calls):
    """The hardware's 2^x is low by 3.4e-9 of its value in the mean; a row's sum may carry that once, however many lanes, waves and
    workgroups share the row.  The bar on the mean error of a token: 5e-9, and three times what the mean of n errors of 6e-8
    (one half step) scatters by."""
    errors = []
    for seed in range(calls):
        g = torch.Generator(device="cuda").manual_seed(seed)
        z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
        t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
        want = torch.cat([torch.log_softmax(z[a:a + 256].double(), 1).gather(1, t[a:a + 256].long()[:, None])[:, 0] for a in range(0, rows, 256)])
        reference = want.float()
        starts = torch.arange(0, rows + 1, 2, dtype=torch.int32, device="cuda")
        _, _, scores = ops.preference_grad(z, t, starts, ref_logp=reference)
        errors.append(scores.double() - (want - reference.double())[0::2])
    errors = torch.cat(errors)
    assert abs(float(errors.mean())) <= 5e-9 + 3 * ref.HALF_STEP / len(errors) ** 0.5
    assert float(errors.square().mean().sqrt()) <= ref.HALF_STEP


@pytest.mark.parametrize("rows,cols", [(40, 13), (40, 8192), (40, 50021), (300, 50021), (40, 151936), (300, 151936), (3, 1300003)])
@pytest.mark.parametrize("odds", [9.2, 4.6])
def test_a_token_that_is_nearly_certain(ops, rows, cols, odds):
    """p = 1 - 1e-4 and 0.99 of one entry, wherever in its row it lies: -logp = log(1 + S) with S the others' share, so a sum whose largest
    term is exactly 1 is off by what its additions round, 2^-24 at most each beside that 1: those of its lane, of its wave (6) and of
    the workgroup and the runs (24 at most).  The bar counts them all where they are few, and 94 where a lane has more than 64 in
    two levels.  Rounding errors of a step of 2^-23 have the standard deviation 2^-23 / sqrt(12) = 0.58 * 2^-24 each, n of them sqrt(n)
    times that, and from 40 rows that is known to a third (1.4 of it is the bar)."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    z = torch.empty(rows, cols, device="cuda").normal_(0, 1, generator=g)
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[:4] = torch.tensor([0, cols - 1, cols // 2, 3], device="cuda")[:min(4, rows)]
    z.scatter_(1, t.long()[:, None], -float("inf"))
    z.scatter_(1, t.long()[:, None], torch.logsumexp(z.double(), 1)[:, None].float() + odds)
    want = torch.log_softmax(z.double(), 1).gather(1, t.long()[:, None])[:, 0]
    assert ((want + float(np.log1p(np.exp(-odds)))).abs() < 1e-5).all()
    n = min(-(-cols // row_lanes(rows, cols)) + 34, 94)
    got, _, _ = ops.token_logprobs(z, t)
    assert ((got.double() - want).abs() <= ref.HALF_STEP * (n + want.abs())).all()
    rms = 1.4 * 0.58 * n ** 0.5 * ref.HALF_STEP
    assert float((got.double() - want).square().mean().sqrt()) <= rms
    if rows % 4 == 0:
        starts = torch.arange(0, rows + 1, 2, dtype=torch.int32, device="cuda")
        _, _, scores = ops.preference_grad(z, t, starts)
        assert float((scores.double() - want[0::2]).square().mean().sqrt()) <= rms
