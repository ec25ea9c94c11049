"""Whole training steps on the other objectives (policy, preference, distillation) and the log-probability pass that feeds
them: losses and gradients against a float64 autograd statement of model and objective, as a run of them is used.
Bars as in test_gpu_step.py: |got - ref| <= 1e-5 + 1e-4 |ref| per tensor, the loss to 1e-5."""
import numpy as np
import pytest
import torch

from tests import refmodel
from tests.test_gpu_step import check_tensors, init_params, rng, tensor_slices

pytestmark = pytest.mark.gpu

MODEL = dict(hidden=64, layers=2, heads=4, kv_heads=2, head_dim=32, ffn=96, vocab=101)
LONG = dict(MODEL, layers=1, vocab=33001)                        # rows shared out between workgroups, not a multiple of four
STARTS = np.array([0, 17, 18, 40, 52], np.int32)                 # one sequence of a single token


@pytest.fixture(scope="module")
def tr():
    from seraph_amd import trainer
    return trainer


def logits_of(cfg, P, tokens, starts, lora=None):
    T = len(tokens)
    seq_id = np.searchsorted(starts, np.arange(T), side="right") - 1
    pos = np.arange(T) - starts[seq_id]
    H, KVH, D = cfg.heads, cfg.kv_heads, cfg.head_dim
    s = cfg.lora_alpha / cfg.lora_rank if cfg.lora_rank else 0.0

    def proj(x, W, ad):
        y = x @ W.T
        return y if ad is None else y + ((x.detach() @ ad[0].T) * s) @ ad[1].T
    x = P["embed"][torch.from_numpy(tokens).long()]
    for l, W in enumerate(P["layers"]):
        ad = lora[l] if lora is not None else {}
        xn = refmodel.rmsnorm(x, W["in_norm"], cfg.rms_eps)
        q = refmodel.rope(proj(xn, W["q"], ad.get("q")), pos, H, D, cfg.rope_theta)
        k = refmodel.rope(proj(xn, W["k"], ad.get("k")), pos, KVH, D, cfg.rope_theta)
        a = refmodel.attention(q, k, proj(xn, W["v"], ad.get("v")), seq_id, H, KVH, D)
        x = x + proj(a, W["o"], ad.get("o"))
        xn = refmodel.rmsnorm(x, W["post_norm"], cfg.rms_eps)
        x = x + proj(torch.nn.functional.silu(proj(xn, W["gate"], ad.get("gate"))) * proj(xn, W["up"], ad.get("up")), W["down"], ad.get("down"))
    return refmodel.rmsnorm(x, P["final_norm"], cfg.rms_eps) @ P["embed"].T


def setup(tr, orc, shape, seed, **lora):
    ocfg = orc.make_config(**shape, rms_eps=1e-5, rope_theta=10000.0, **lora)
    cfg = tr.model_config(**shape, rms_eps=1e-5, rope_theta=10000.0, **lora)
    p = init_params(orc, ocfg, seed)
    T = int(STARTS[-1])
    tok = rng(seed + 1).integers(0, shape["vocab"], T).astype(np.int32)
    t = tr.Trainer(cfg, tr.optim_config(3.14e-4), max_tokens=T, max_batch=len(STARTS) - 1)
    t.upload(tr.PARAMS, p)
    return ocfg, p, tok, t


def live_rows(T, keep):
    live = np.ones(T, bool)
    live[STARTS[1:] - 1] = False
    return torch.from_numpy(live & (keep != 0))


def next_tokens(tok):
    nxt = np.zeros(len(tok), np.int64)
    nxt[:-1] = tok[1:]
    return torch.from_numpy(nxt)


def policy_loss(lsm, nxt, live, a):
    logp = lsm[torch.arange(len(nxt)), nxt]
    ratio = torch.exp(logp - a["old"])
    loss = -torch.minimum(ratio * a["adv"], torch.clamp(ratio, 0.8, 1.25) * a["adv"])
    d = a["ref"] - logp
    ent = -(lsm.exp() * lsm).sum(1)
    return ((loss + 0.05 * (torch.exp(d) - d - 1) - 0.01 * ent) * a["w"])[live].sum() / live.sum()


def preference_loss(lsm, nxt, live, a):
    d = torch.where(live, lsm[torch.arange(len(nxt)), nxt] - a["ref"], 0.0)
    s = torch.stack([d[x:y].sum() for x, y in zip(STARTS[:-1], STARTS[1:])])
    h = 0.4 * (s[0::2] - s[1::2])
    return (-0.9 * torch.nn.functional.logsigmoid(h) - 0.1 * torch.nn.functional.logsigmoid(-h)).mean(), s


def distill_loss(logits, nxt, live, a):
    lp = torch.log_softmax(logits / 2.0, 1).gather(1, a["ids"])
    lq = torch.log_softmax(a["teacher"] / 2.0, 1)
    kl = (lq.exp() * (lq - lp)).sum(1)
    hard = -torch.log_softmax(logits, 1)[torch.arange(len(nxt)), nxt]
    return ((2.8 * kl + 0.3 * hard) * a["w"])[live].sum() / live.sum()


@pytest.mark.parametrize("shape", [MODEL, LONG])
def test_full_steps_on_each_objective(tr, orc, shape):
    ocfg, p, tok, t = setup(tr, orc, shape, 11)
    T, V = len(tok), shape["vocab"]
    r = rng(12)
    flat = torch.tensor(p, dtype=torch.float64, requires_grad=True)
    logits = logits_of(ocfg, refmodel.split_params(ocfg, flat), tok, STARTS)
    lsm = torch.log_softmax(logits, 1)
    nxt = next_tokens(tok)
    w = r.choice([0.0, 0.5, 1.5], T).astype(np.float32)
    live = live_rows(T, w)
    inner = live_rows(T, np.ones(T)).numpy()

    # the pass that the other steps take their inputs from
    logp, entropy = t.token_logprobs(tok, STARTS, want_entropy=True)
    want = lsm.detach()[torch.arange(T), nxt].numpy()
    ent = -(lsm.exp() * lsm).sum(1).detach().numpy()
    assert np.abs(logp[inner] - want[inner]).max() <= 1e-5 + 1e-4 * np.abs(want).max() and (logp[~inner] == 0).all()
    assert np.abs(entropy[inner] - ent[inner]).max() <= 1e-5 + 1e-4 * ent.max() and (entropy[~inner] == 0).all()
    assert (t.download(tr.PARAMS) == p).all() and t.optimizer_step == 0

    adv, old, ref = r.standard_normal(T).astype(np.float32), (want - 0.07).astype(np.float32), (want + 0.2 * r.standard_normal(T)).astype(np.float32)
    ids = np.stack([r.permutation(V)[:9] for _ in range(T)]).astype(np.uint32)
    teacher = (2 * r.standard_normal((T, 9))).astype(np.float16)
    d64 = lambda a: torch.from_numpy(np.asarray(a, np.float64))          # noqa: E731
    arrays = dict(adv=d64(adv), old=d64(old), ref=d64(ref), w=d64(w), ids=torch.from_numpy(ids.astype(np.int64)), teacher=d64(teacher))
    pl, scores = preference_loss(lsm, nxt, live, arrays)
    sl = tensor_slices(ocfg)
    steps = [
        (policy_loss(lsm, nxt, live, arrays), lambda run: t.step_policy(tok, STARTS, adv, old, ref_logp=ref, weights=w, clip=(0.2, 0.25), kl_coef=0.05,
                                                                        entropy_coef=0.01, run_optimizer=run)),
        (pl, lambda run: t.step_preference(tok, STARTS, supervised=w, ref_logp=ref, beta=0.4, label_smoothing=0.1, run_optimizer=run)[0]),
        (distill_loss(logits, nxt, live, arrays), lambda run: t.step_distill(tok, STARTS, ids, teacher, weights=w, temperature=2.0, soft_coef=2.8,
                                                                             hard_coef=0.3, run_optimizer=run))]
    for want_loss, step in steps:
        g, = torch.autograd.grad(want_loss, flat, retain_graph=True)
        loss = step(False)
        assert abs(loss - want_loss.item()) <= 1e-5 * max(1.0, abs(want_loss.item()))
        check_tensors(t.download(tr.GRADS), g.numpy(), sl, "grad")
    _, got = t.step_preference(tok, STARTS, supervised=w, ref_logp=ref, beta=0.4, label_smoothing=0.1, run_optimizer=False)
    assert np.abs(got - scores.detach().numpy()).max() <= 1e-4
    # the cross entropy step between them is what it was before
    ref_loss, ref_g = orc.step_full(ocfg, p, tok, STARTS)
    assert abs(t.step(tok, STARTS, run_optimizer=False) - ref_loss) < 1e-5 * max(1.0, abs(ref_loss))
    check_tensors(t.download(tr.GRADS), ref_g, sl, "grad")
    assert (t.download(tr.PARAMS) == p).all()
    # the optimizer runs behind an objective as behind the cross entropy
    g, = torch.autograd.grad(steps[2][0], flat)
    steps[2][1](True)
    assert t.optimizer_step == 1
    z = np.zeros_like(p)
    rw, _, _ = orc.adamw(p, g.numpy().astype(np.float32), z, z, orc.lr_schedule(3.14e-4, 1, 1), 0.9, 0.999, 0.01, 1e-8, 1)
    check_tensors(t.download(tr.PARAMS), rw, sl, "weight")
    t.close()


def test_lora_preference_against_its_own_base(tr, orc):
    """The frozen base model of the adapters being trained is the reference: one trainer, two passes, one step."""
    lora = dict(lora_rank=4, lora_alpha=8.0, lora_mask=0b1111111)
    ocfg, p, tok, t = setup(tr, orc, MODEL, 21, **lora)
    T = len(tok)
    ad = (0.05 * rng(22).standard_normal(t.nlora)).astype(np.float32)
    t.upload(tr.LORA_PARAMS, ad)
    P = refmodel.split_params(ocfg, torch.tensor(p, dtype=torch.float64))
    flat = torch.tensor(ad, dtype=torch.float64, requires_grad=True)
    nxt, inner = next_tokens(tok), live_rows(T, np.ones(T))
    base = torch.log_softmax(logits_of(ocfg, P, tok, STARTS), 1)[torch.arange(T), nxt]
    lsm = torch.log_softmax(logits_of(ocfg, P, tok, STARTS, refmodel.split_lora(ocfg, flat)), 1)
    ref = t.token_logprobs(tok, STARTS, adapters=False)
    now = t.token_logprobs(tok, STARTS)
    own = lsm.detach()[torch.arange(T), nxt].numpy()
    keep = inner.numpy()
    assert np.abs(ref[keep] - base.numpy()[keep]).max() <= 1e-5 + 1e-4 * np.abs(own).max()
    assert np.abs(now[keep] - own[keep]).max() <= 1e-5 + 1e-4 * np.abs(own).max()
    assert np.abs(ref - now).max() > 1e-3                        # the adapters do something
    want, scores = preference_loss(lsm, nxt, inner, dict(ref=torch.from_numpy(ref.astype(np.float64))))
    g, = torch.autograd.grad(want, flat)
    loss, got = t.step_preference(tok, STARTS, ref_logp=ref, beta=0.4, label_smoothing=0.1, run_optimizer=False)
    assert abs(loss - want.item()) <= 1e-5 and np.abs(got - scores.detach().numpy()).max() <= 1e-4
    grads = t.download(tr.LORA_GRADS).astype(np.float64)
    assert (np.abs(grads - g.numpy()) <= 1e-5 + 1e-4 * np.abs(g.numpy())).all()
    t.step_preference(tok, STARTS, ref_logp=ref, beta=0.4, label_smoothing=0.1)
    assert t.optimizer_step == 1 and (t.download(tr.LORA_PARAMS) != ad).any()
    assert np.array_equal(t.token_logprobs(tok, STARTS, adapters=False), ref)      # the base has not moved
    t.close()


def test_objective_accumulates_with_the_cross_entropy(tr, orc):
    """A gradient accumulation window of one distillation and one cross entropy step: the sum of both gradients."""
    ocfg, p, tok, t = setup(tr, orc, MODEL, 31)
    t.close()
    T = len(tok)
    t = tr.Trainer(tr.model_config(**MODEL, rms_eps=1e-5, rope_theta=10000.0), tr.optim_config(1e-3, gradient_accumulation_steps=2), max_tokens=T, max_batch=4)
    t.upload(tr.PARAMS, p)
    r = rng(32)
    ids = np.stack([r.permutation(101)[:5] for _ in range(T)]).astype(np.uint32)
    teacher = r.standard_normal((T, 5)).astype(np.float32)
    flat = torch.tensor(p, dtype=torch.float64, requires_grad=True)
    logits = logits_of(ocfg, refmodel.split_params(ocfg, flat), tok, STARTS)
    w = np.ones(T, np.float32)
    arrays = dict(ids=torch.from_numpy(ids.astype(np.int64)), teacher=torch.from_numpy(teacher.astype(np.float64)), w=torch.ones(T, dtype=torch.float64))
    g, = torch.autograd.grad(distill_loss(logits, next_tokens(tok), live_rows(T, w), arrays), flat)
    t.step_distill(tok, STARTS, ids, teacher, temperature=2.0, soft_coef=2.8, hard_coef=0.3)
    assert t.optimizer_step == 0
    _, both = orc.step_full(ocfg, p, tok, STARTS, grads0=g.numpy().astype(np.float32))
    t.step(tok, STARTS)
    assert t.optimizer_step == 1
    check_tensors(t.download(tr.GRADS), both, tensor_slices(ocfg), "accumulated grad")
    t.close()


def test_batches_without_a_prediction_and_refusals(tr, orc, capfd):
    from seraph_amd._lib import SeraphError
    ocfg, p, tok, t = setup(tr, orc, MODEL, 41)
    T = len(tok)
    f, ids = np.zeros(T, np.float32), np.zeros((T, 2), np.uint32)
    assert t.step_policy(tok, STARTS, f, f, weights=f) == 0.0
    assert t.step_distill(tok, STARTS, ids, np.zeros((T, 2), np.float32), weights=f) == 0.0
    assert t.optimizer_step == 0 and (t.download(tr.PARAMS) == p).all()
    loss, scores = t.step_preference(tok, STARTS, supervised=f, beta=0.5, run_optimizer=False)
    assert abs(loss - np.log(2)) < 1e-6 and (scores == 0).all() and (t.download(tr.GRADS) == 0).all()
    ones = np.arange(T + 1, dtype=np.int32)
    assert (t.token_logprobs(tok[:4], ones[:5]) == 0).all()              # sequences of one token: nothing is predicted
    for bad in (lambda: t.step_policy(tok, STARTS, f[:-1], f), lambda: t.step_policy(tok, STARTS, f, f, kl_coef=0.1),
                lambda: t.step_policy(tok, STARTS, f, f, clip=(-0.1, 0.2)), lambda: t.step_preference(tok, STARTS[:-1]),
                lambda: t.step_preference(tok, STARTS, kind="other"), lambda: t.step_preference(tok, STARTS, beta=0.0),
                lambda: t.step_preference(tok, None), lambda: t.step_distill(tok, STARTS, ids[:, 0], f),
                lambda: t.step_distill(tok, STARTS, np.zeros((T, 1025), np.uint32), np.zeros((T, 1025), np.float32)),
                lambda: t.step_distill(tok, STARTS, ids, np.zeros((T, 2), np.float32), temperature=0.0),
                lambda: t.token_logprobs(tok[:1]), lambda: t.token_logprobs(np.zeros(2 * T, np.int32))):
        with pytest.raises(SeraphError):
            bad()
    assert (t.download(tr.PARAMS) == p).all()
    ref_loss, _ = orc.step_full(ocfg, p, tok, STARTS)                    # a refused step leaves a trainer that works
    assert abs(t.step(tok, STARTS, run_optimizer=False) - ref_loss) < 1e-5 * max(1.0, abs(ref_loss))
    capfd.readouterr()
    t.enable_nan_check()
    t.set_nan_dump_prefix(None)
    assert np.isnan(t.step_policy(tok, STARTS, np.full(T, np.nan, np.float32), f)) and t.nan_detected
    assert (t.download(tr.PARAMS) == p).all()
    t.close()


def test_pairs_of_single_tokens(tr, orc):
    """Nothing is predicted anywhere: the loss of equal scores, no gradient, and the step counts as one."""
    _, p, tok, t = setup(tr, orc, MODEL, 47)
    ones = np.arange(5, dtype=np.int32)
    loss, scores = t.step_preference(tok[:4], ones, kind="hinge", beta=0.5, margin=0.25, run_optimizer=False)
    assert loss == 1.25 and (scores == 0).all() and (t.download(tr.GRADS) == 0).all()
    loss, scores = t.step_preference(tok[:4], ones, beta=0.5)
    assert abs(loss - np.log(2)) < 1e-6 and (scores == 0).all() and t.optimizer_step == 1
    t.close()
