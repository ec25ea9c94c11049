"""Steps of a LoRA trainer on the policy and the distillation objective, and the teacher's types and own logsumexp as a step takes
them, against a float64 autograd statement of model and objective.  Bars as in test_gpu_objective_steps.py."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import refmodel
from tests.test_gpu_objective_steps import MODEL, STARTS, live_rows, logits_of, next_tokens, policy_loss, setup, tr      # noqa: F401
from tests.test_gpu_step import check_tensors, rng, tensor_slices

pytestmark = pytest.mark.gpu

LORA = dict(lora_rank=4, lora_alpha=8.0, lora_mask=0b1111111)


def f64(a):
    return torch.from_numpy(np.asarray(a, np.float64))


def lora_setup(tr, orc, seed):      # noqa: F811
    ocfg, p, tok, t = setup(tr, orc, MODEL, seed, **LORA)
    ad = (0.05 * rng(seed + 1).standard_normal(t.nlora)).astype(np.float32)
    t.upload(tr.LORA_PARAMS, ad)
    flat = torch.tensor(ad, dtype=torch.float64, requires_grad=True)
    P = refmodel.split_params(ocfg, torch.tensor(p, dtype=torch.float64))
    return ocfg, tok, t, flat, logits_of(ocfg, P, tok, STARTS, refmodel.split_lora(ocfg, flat))


def check_step(tr, t, want, flat, loss):      # noqa: F811
    g, = torch.autograd.grad(want, flat, retain_graph=True)
    assert abs(loss - want.item()) <= 1e-5 * max(1.0, abs(want.item()))
    grads = t.download(tr.LORA_GRADS).astype(np.float64)
    assert np.abs(g.numpy()).max() > 1e-3 and (np.abs(grads - g.numpy()) <= 1e-5 + 1e-4 * np.abs(g.numpy())).all()


def own_lse_loss(logits, nxt, live, a, temperature, soft, hard):
    lp = torch.log_softmax(logits / temperature, 1).gather(1, a["ids"])
    lq = a["teacher"] / temperature - a["lse"][:, None]
    kl = (lq.exp() * (lq - lp)).sum(1)
    label = -torch.log_softmax(logits, 1)[torch.arange(len(nxt)), nxt]
    return ((soft * kl + hard * label) * a["w"])[live].sum() / live.sum()


def test_lora_steps_on_policy_and_distillation(tr, orc):      # noqa: F811
    ocfg, tok, t, flat, logits = lora_setup(tr, orc, 61)
    T, V, r = len(tok), MODEL["vocab"], rng(63)
    w = r.choice([0.0, 0.5, 1.5], T).astype(np.float32)
    live, nxt = live_rows(T, w), next_tokens(tok)
    lsm = torch.log_softmax(logits, 1)
    now = lsm.detach()[torch.arange(T), nxt].numpy()
    adv, old, ref = r.standard_normal(T).astype(np.float32), (now - 0.07).astype(np.float32), (now + 0.2 * r.standard_normal(T)).astype(np.float32)
    arrays = dict(adv=f64(adv), old=f64(old), ref=f64(ref), w=f64(w))
    loss = t.step_policy(tok, STARTS, adv, old, ref_logp=ref, weights=w, clip=(0.2, 0.25), kl_coef=0.05, entropy_coef=0.01, run_optimizer=False)
    check_step(tr, t, policy_loss(lsm, nxt, live, arrays), flat, loss)

    ids = np.stack([r.permutation(V)[:7] for _ in range(T)]).astype(np.uint32)
    teacher = (2 * r.standard_normal((T, 7))).astype(np.float32)
    lse = (np.log(np.exp(teacher / 1.5).sum(1)) + 0.3 * r.random(T)).astype(np.float32)      # the list is most of the distribution
    arrays.update(ids=torch.from_numpy(ids.astype(np.int64)), lse=f64(lse), teacher=f64(teacher))
    kw = dict(temperature=1.5, soft_coef=2.0, hard_coef=0.3, weights=w, teacher_lse=lse)
    loss = t.step_distill(tok, STARTS, ids, teacher, run_optimizer=False, **kw)
    want = own_lse_loss(logits, nxt, live, arrays, 1.5, 2.0, 0.3)
    check_step(tr, t, want, flat, loss)
    before = t.download(tr.LORA_PARAMS)
    t.step_distill(tok, STARTS, ids, teacher, **kw)
    assert t.optimizer_step == 1 and (t.download(tr.LORA_PARAMS) != before).any()
    t.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("top_k", [1, 7, 300])
def test_the_teachers_types_through_the_step(tr, orc, dtype, top_k):      # noqa: F811
    """All three types as the C interface takes them, lists longer than the vocabulary among them."""
    from seraph_amd._lib import DistillOptions
    from seraph_amd.trainer import _lib
    ocfg, p, tok, t = setup(tr, orc, MODEL, 71)
    T, V, r = len(tok), MODEL["vocab"], rng(73)
    ids = r.integers(0, V, (T, top_k)).astype(np.uint32)
    teacher = torch.from_numpy((2 * r.standard_normal((T, top_k))).astype(np.float32)).to(dtype)
    held = teacher.contiguous().view(torch.int32 if dtype == torch.float32 else torch.int16).numpy()
    flat = torch.tensor(p, dtype=torch.float64, requires_grad=True)
    logits = logits_of(ocfg, refmodel.split_params(ocfg, flat), tok, STARTS)
    live = live_rows(T, np.ones(T))
    arrays = dict(ids=torch.from_numpy(ids.astype(np.int64)), teacher=teacher.double(), w=torch.ones(T, dtype=torch.float64),
                  lse=torch.logsumexp(teacher.double(), 1))
    want = own_lse_loss(logits, next_tokens(tok), live, arrays, 1.0, 1.0, 0.0)
    g, = torch.autograd.grad(want, flat)
    loss = C.c_float()
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    rc = _lib().hip_train_step_distill(t._h, tok.ctypes.data, T, STARTS.ctypes.data, len(STARTS) - 1, ids.ctypes.data, held.ctypes.data, None, top_k,
                                       None, DistillOptions(1.0, 1.0, 0.0, code), 0, C.byref(loss))
    assert rc == 0 and abs(loss.value - want.item()) <= 1e-5 * max(1.0, abs(want.item()))
    check_tensors(t.download(tr.GRADS), g.numpy(), tensor_slices(ocfg), "grad")
    t.close()


def test_offsets_that_do_not_fit_are_refused_whatever_counts(tr, orc):      # noqa: F811
    """Also where no prediction would count: an empty sequence among as many sequences as tokens is no batch without predictions."""
    from seraph_amd._lib import SeraphError
    ocfg, p, tok, t = setup(tr, orc, MODEL, 81)
    T = len(tok)
    f, ids, z = np.zeros(T, np.float32), np.zeros((T, 2), np.uint32), np.zeros((T, 2), np.float32)
    short = np.array([0, 1, 1, 2, 4], np.int32)                   # tokens 2 and 3 are one sequence, which has a prediction
    for starts in (short, np.array([0, 2, 1, 4], np.int32), np.array([0, 1, 2, 3], np.int32), np.array([1, 2, 3, 4], np.int32)):
        for call in (lambda s: t.token_logprobs(tok[:4], s), lambda s: t.step_policy(tok[:4], s, f[:4], f[:4], weights=f[:4]),
                     lambda s: t.step_distill(tok[:4], s, ids[:4], z[:4], weights=f[:4])):
            with pytest.raises(SeraphError):
                call(starts)
    with pytest.raises(SeraphError):
        t.step_preference(tok[:4], short, supervised=f[:4])
    assert (t.token_logprobs(tok[:4], np.arange(5, dtype=np.int32)) == 0).all()
    assert (t.download(tr.PARAMS) == p).all() and t.optimizer_step == 0
    t.close()


def test_offsets_past_the_batch_are_refused_before_use(tr, orc):      # noqa: F811
    """In the middle of the offsets too, where first and last fit: the host's staging room ends with the batch."""
    from seraph_amd._lib import SeraphError
    ocfg, p, tok, t = setup(tr, orc, MODEL, 91)
    T = len(tok)
    f = np.ones(T, np.float32)
    for middle in ([1 << 20], [2, 1 << 30], [1 << 28, 5]):
        starts = np.array([0] + middle + [T], np.int32)
        assert t.eval_forward(tok, starts) == -1.0
        for call in (lambda: t.step(tok, starts), lambda: t.token_logprobs(tok, starts), lambda: t.step_policy(tok, starts, f, f)):
            with pytest.raises(SeraphError):
                call()
    ref_loss, _ = orc.step_full(ocfg, p, tok, STARTS)
    assert abs(t.step(tok, STARTS, run_optimizer=False) - ref_loss) < 1e-5 * max(1.0, abs(ref_loss))
    t.close()


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
def test_a_checked_preference_step_stops_at_a_pair_without_a_score(tr, orc, kind):      # noqa: F811
    """NaN in ref_logp, all logits finite: the check finds it in the logits' gradient and no weight moves."""
    ocfg, p, tok, t = setup(tr, orc, MODEL, 101)
    ref = np.full(len(tok), -4.0, np.float32)
    t.enable_nan_check()
    t.set_nan_dump_prefix(None)
    loss, _ = t.step_preference(tok, STARTS, ref_logp=ref, kind=kind, beta=0.3, run_optimizer=False)
    assert np.isfinite(loss) and not t.nan_detected
    ref[20] = np.nan                                              # a supervised token of the second pair
    loss, _ = t.step_preference(tok, STARTS, ref_logp=ref, kind=kind, beta=0.3)
    assert np.isnan(loss) and t.nan_detected
    assert (t.download(tr.PARAMS) == p).all()
    t.close()
