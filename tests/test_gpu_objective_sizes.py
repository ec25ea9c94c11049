"""The objectives over logits at the ends of the sizes they take: as many rows as a call holds, the widest row, and the forms of long
batches captured into a graph."""
import numpy as np
import pytest
import torch

from tests import objectives_ref as ref
from tests.test_gpu_objectives import dev, make, ops, policy_inputs      # noqa: F401

pytestmark = pytest.mark.gpu


def test_as_many_rows_as_a_call_holds(ops):
    """2^24 - 1 rows of three columns, against a softmax in 64 bits by torch; bounds as in objectives_ref.unit()."""
    rows, cols = (1 << 24) - 1, 3
    g = torch.Generator(device="cuda").manual_seed(24)
    z = torch.empty(rows, cols, device="cuda").normal_(generator=g)
    t = torch.randint(0, cols + 1, (rows,), device="cuda", generator=g, dtype=torch.int32)
    live = t < cols
    lsm = torch.log_softmax(z.double(), 1)
    hot = torch.zeros_like(lsm).scatter_(1, t.long().clamp(max=cols - 1)[:, None], 1.0)
    want = (lsm * hot).sum(1)
    spread = (z.amax(1) - z.amin(1)).double()
    u = ref.HALF_STEP * (6.0 * spread + cols / 64.0 + 40.0)
    logp, lse, _ = ops.token_logprobs(z, t, want_lse=True)
    assert (logp[~live] == 0).all() and ((logp.double() - want).abs() <= u + ref.HALF_STEP * want.abs())[live].all()
    p = lsm.exp()
    one = torch.ones(rows, device="cuda")
    old = (want - 0.1).float()
    grad, loss, _, _, _ = ops.policy_grad(z, t, one, old, rows)
    f = torch.where(live, torch.exp(want - old.double()) / rows, 0.0)[:, None]
    assert ((grad.double() - f * (p - hot)).abs() <= 4 * u[:, None] * f * (p + hot) + 1e-38).all() and (loss[~live] == 0).all()
    ids = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    grad, loss = ops.distill_grad(z, ids, one[:, None].contiguous(), rows)
    first = torch.tensor([1.0, 0.0, 0.0], dtype=torch.float64, device="cuda")
    assert ((grad.double() - (p - first) / rows).abs() <= 4 * u[:, None] * (p + first) / rows).all()
    assert ((loss.double() + lsm[:, 0]).abs() <= 4 * u * (1 + lsm[:, 0].abs())).all()


def test_the_widest_row(ops):
    """2^31 - 1 columns: some of mass at the ends and around powers of two, -40 everywhere else."""
    cols = (1 << 31) - 1
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    at = torch.tensor([0, 1, 31, 1 << 20, (1 << 29) - 1, 1 << 29, (1 << 30) + 5, cols - 5, cols - 2, cols - 1], device="cuda")
    high = torch.linspace(-1.0, 2.0, len(at), dtype=torch.float64, device="cuda").float()
    other = (cols - len(at)) * float(np.exp(-40.0))
    lse = float(torch.log(high.double().exp().sum() + other))
    logp = high.double() - lse
    z = torch.full((2, cols), -40.0, device="cuda")
    z[:, at] = high
    # six steps of the exponentials' arguments (42 at most), the additions that matter (few entries have mass)
    u = ref.HALF_STEP * (6 * 42 + 64)

    def check_row(grad, factor, hot):
        """factor (hot - p), hot {column: mass}, total mass 1; the row is overwritten"""
        want = -factor * torch.exp(logp)
        for c, q in hot.items():
            want[c] += factor * q
        assert ((grad[at].double() - want).abs() <= 4 * u * abs(factor)).all()
        grad[at] = 0.0
        top = max(abs(float(grad.max())), abs(float(grad.min())))
        assert 0 < top <= 1.001 * abs(factor) * float(np.exp(-40.0 - lse))

    for i in range(0, len(at), 3):
        t = at[[i, i]].to(torch.int32)
        got, norm, _ = ops.token_logprobs(z, t, want_lse=True)
        assert abs(float(got[0]) - float(logp[i])) <= u + ref.HALF_STEP * abs(float(logp[i])) and abs(float(norm[1]) - lse) <= u + ref.HALF_STEP * abs(lse)
    i = len(at) - 1
    t = at[[i, 0]].to(torch.int32)
    one = torch.ones(2, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    grad = torch.empty_like(z)
    ops.policy_grad(z, t, one, logp[[i, 0]].float(), 1, grad=grad)
    check_row(grad[0], -1.0, {i: 1.0})
    check_row(grad[1], -1.0, {0: 1.0})
    ids = at[[i, 3]].to(torch.int32).repeat(2, 1)
    ops.distill_grad(z, ids, torch.zeros(2, 2, device="cuda"), 1, grad=grad)
    check_row(grad[1], -1.0, {i: 0.5, 3: 0.5})
    starts = torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
    _, loss, scores = ops.preference_grad(z, t, starts, kind="hinge", beta=0.25, grad=grad)
    assert abs(float(scores[0]) - float(logp[i])) <= u + ref.HALF_STEP * abs(float(logp[i])) and float(scores[1]) == 0 and float(loss[0]) > 1
    assert not grad[1].any()
    check_row(grad[0], -0.25, {i: 1.0})


@pytest.mark.parametrize("rows,cols", [(1300, 50), (300, 40001)])
def test_long_batches_captured_and_replayed(ops, rows, cols):
    """Pairs of their own kernel, runs that are joined, and gradients over the logits, captured; each replay on new logits against the
    eager result, with eager work in between."""
    r, z, t = make(rows, cols, cols + 71)
    adv, old, refl = policy_inputs(r, z, t)
    starts = np.linspace(0, rows, 5).astype(np.uint32)
    Z, T, A, O, R, S = (dev(a) for a in (z, t, adv, old, refl, starts))
    W = torch.empty_like(Z)

    def over(call):
        W.copy_(Z)
        return call(W)
    calls = (lambda: ops.preference_grad(Z, T, S, ref_logp=R), lambda: over(lambda w: ops.preference_grad(w, T, S, ref_logp=R, grad=w)),
             lambda: ops.token_logprobs(Z, T, seq_starts=S, want_lse=True, want_entropy=True),
             lambda: over(lambda w: ops.policy_grad(w, T, A, O, rows, ref_logp=R, kl_coef=0.1, seq_starts=S, grad=w)))
    for call in calls:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        for k in range(3):
            Z.copy_(dev((2 * np.random.default_rng(200 + k).standard_normal((rows, cols))).astype(np.float32)))
            want = [None if a is None else a.clone() for a in call()]
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert (a is None and b is None) or torch.equal(a, b)
