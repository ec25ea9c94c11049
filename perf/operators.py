"""What is measured of the objectives over vocabulary logits: token log-probabilities, the clipped policy loss, the paired
preference loss and distillation from a teacher's top logits.

A training step of the framework ends its forward pass with FP32 logits [rows, vocab]; each of these operators turns them
into a loss and (all but the first) the gradient with respect to them.  `run` computes them in their plain form, or, with
`own`, by the calls that a user makes.
"""
import math
import random

import torch

own = False

CARD_CASE = 4096 * 151936      # elements of the largest logits that a case here has

# The vocabularies: 8192 and 151936 are the configurations that the framework's benchmark trains, 50021 stands for a
# vocabulary that is not a multiple of anything, 32000 for the common middle.


def listed():
    return [
        # eight sequences scored by one token each: the step where launches count, not bytes
        dict(name="logprobs-8x151936", op="logprobs", rows=8, vocab=151936, seqs=0, prompt=0.0, entropy=False),
        # log-probabilities and entropies of the rollouts of a small model, 8 x 256 tokens
        dict(name="logprobs-2048x8192", op="logprobs", rows=2048, vocab=8192, seqs=8, prompt=0.25, entropy=True),
        # the reference model's pass over a batch of two 2048-token sequences
        dict(name="logprobs-4096x151936", op="logprobs", rows=4096, vocab=151936, seqs=2, prompt=0.0, entropy=False),
        # a policy step of the small model, 8 x 256 tokens, with an entropy bonus
        dict(name="policy-2048x8192", op="policy", rows=2048, vocab=8192, seqs=8, prompt=0.25, entropy=True, kl=True),
        # short answers over an odd vocabulary, one advantage for each token, no reference model
        dict(name="policy-777x50021", op="policy", rows=777, vocab=50021, seqs=5, prompt=0.1, entropy=False, kl=False),
        # a policy step of the 151936-token vocabulary with the KL term, prompts masked
        dict(name="policy-4096x151936", op="policy", rows=4096, vocab=151936, seqs=8, prompt=0.1, entropy=False, kl=True),
        # one pair of short answers of the small model
        dict(name="preference-96x8192", op="preference", rows=96, vocab=8192, seqs=2, prompt=0.2, kind="sigmoid", average=False),
        # three pairs of ragged lengths over an odd vocabulary, averaged over the tokens of an answer
        dict(name="preference-1531x50021", op="preference", rows=1531, vocab=50021, seqs=6, prompt=0.1, kind="squared", average=True),
        # four pairs of about 512 tokens a side, the LoRA model's vocabulary
        dict(name="preference-4096x151936", op="preference", rows=4096, vocab=151936, seqs=8, prompt=0.1, kind="sigmoid", average=False),
        # a small batch of the small model, 32 listed logits for each token
        dict(name="distill-256x8192", op="distill", rows=256, vocab=8192, seqs=1, prompt=0.0, top_k=32, teacher="float32", temperature=1.0, hard=False),
        # a long list of teacher logits, warm distribution, mixed with the labels
        dict(name="distill-2047x32000", op="distill", rows=2047, vocab=32000, seqs=4, prompt=0.1, top_k=256, teacher="bfloat16", temperature=2.0, hard=True),
        # a distillation step of the 151936-token vocabulary
        dict(name="distill-4096x151936", op="distill", rows=4096, vocab=151936, seqs=2, prompt=0.0, top_k=64, teacher="float16", temperature=1.0, hard=False),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "distill"])
    vocab = _between(rng, 1000, 160000)
    if rng.random() < 0.5:
        vocab |= 1
    rows = _between(rng, 1, max(1, min(8192, CARD_CASE // vocab)))
    seqs = rng.choice([0, 1, 2, 3, 8])
    if op == "preference":
        rows, seqs = max(rows, 4), 2 * max(1, min(rng.choice([1, 2, 3, 8]), rows // 8))
    if seqs and rows < 2 * seqs:
        seqs = 0
    case = dict(op=op, rows=rows, vocab=vocab, seqs=seqs, prompt=rng.choice([0.0, 0.1, 0.3]))
    if op == "logprobs":
        case["entropy"] = rng.random() < 0.5
    elif op == "policy":
        case.update(entropy=rng.random() < 0.4, kl=rng.random() < 0.6)
    elif op == "preference":
        case.update(kind=rng.choice(["sigmoid", "hinge", "squared"]), average=rng.random() < 0.5)
    else:
        case.update(top_k=min(_between(rng, 1, 512), vocab // 2), teacher=rng.choice(["float32", "float16", "bfloat16"]),
                    temperature=rng.choice([1.0, 1.0, 2.0, 0.7]), hard=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------ inputs
def _layout(case):
    """(offsets of the packed sequences or None, the rows that are supervised): by the case alone."""
    rows, seqs = case["rows"], case["seqs"]
    if not seqs:
        return None, [True] * rows
    rng = random.Random(rows * 131 + seqs)
    cuts = sorted(rng.sample(range(1, rows // 2), seqs - 1)) if seqs > 1 else []
    starts = [0] + [2 * c for c in cuts] + [rows]                     # ragged, two tokens at least
    live = [False] * rows
    for a, b in zip(starts, starts[1:]):
        first = a + int(case["prompt"] * (b - a))
        for r in range(first, b - 1):                                 # the last token of a sequence has no successor
            live[r] = True
    return starts, live


def _chunks(rows, vocab, elements=1 << 27):
    step = max(1, elements // vocab)
    return [(a, min(rows, a + step)) for a in range(0, rows, step)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    starts, live = _layout(case)
    logits = torch.empty(rows, vocab, device="cuda").normal_(0.0, 2.0, generator=g)
    ids = torch.empty(rows, dtype=torch.int32, device="cuda")
    logp = torch.empty(rows, dtype=torch.float64, device="cuda")
    teacher_ids, teacher_logits = None, None
    if case["op"] == "distill":
        k = case["top_k"]
        teacher_ids = torch.empty(rows, k, dtype=torch.int32, device="cuda")
        teacher_logits = torch.empty(rows, k, dtype=getattr(torch, case["teacher"]), device="cuda")
    for a, b in _chunks(rows, vocab):
        z = logits[a:b]
        noise = torch.empty_like(z).exponential_(generator=g)
        pick = (z - noise.log_()).argmax(1)                           # a token sampled from the model's own distribution
        ids[a:b] = pick.to(torch.int32)
        logp[a:b] = z.gather(1, pick[:, None])[:, 0].double() - torch.logsumexp(z.double(), 1)
        if teacher_ids is not None:                                   # a teacher that mostly agrees with the student
            top = (z + noise.normal_(0.0, 1.0, generator=g)).topk(k, 1)
            teacher_ids[a:b] = top.indices.to(torch.int32)
            teacher_logits[a:b] = top.values.to(teacher_logits.dtype)
    mask = torch.tensor(live, device="cuda")
    ids[~mask] = -1                                                   # no supervision
    state = dict(case=case, logits=logits, ids=ids, valid=max(1, sum(live)), live=mask,
                 starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda"))

    def noisy(std):
        return (logp + torch.empty_like(logp).normal_(0.0, std, generator=g)).float()
    if case["op"] != "logprobs":
        state["grad"] = torch.empty_like(logits)                      # the buffer that a training loop keeps
    if case["op"] == "policy":
        state.update(old=noisy(0.15), ref=noisy(0.3) if case["kl"] else None, kl_coef=0.04 if case["kl"] else 0.0,
                     entropy_coef=0.01 if case["entropy"] else 0.0,
                     advantages=torch.empty(rows, device="cuda").normal_(generator=g))
    if case["op"] == "preference":
        state.update(ref=noisy(0.3), beta=0.1, smoothing=0.05 if case["kind"] == "sigmoid" else 0.0)
    if case["op"] == "distill":
        t = case["temperature"]
        weights = torch.empty(rows, device="cuda").uniform_(0.5, 1.5, generator=g) * mask
        state.update(teacher_ids=teacher_ids, teacher_logits=teacher_logits, weights=weights, temperature=t,
                     soft=0.7 * t * t if case["hard"] else 1.0, hard=0.3 if case["hard"] else 0.0)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return {"logprobs": _logprobs, "policy": _policy, "preference": _preference, "distill": _distill}[state["case"]["op"]](state)


_module = None


def _ops():
    global _module
    if _module is None:
        from seraph_amd import ops
        _module = ops
    return _module


def _plain_stats(z):
    m = z.amax(1, keepdim=True)
    x = z - m
    e = torch.exp(x)
    return m, x, e, e.sum(1, keepdim=True)


def _plain_ids(state):
    """The supervised rows, and an index that stays in range on the others."""
    return state["live"], torch.where(state["live"], state["ids"], 0).long()[:, None]


def _logprobs(state):
    z = state["logits"]
    want = state["case"]["entropy"]
    if own:
        logp, lse, entropy = _ops().token_logprobs(z, state["ids"], seq_starts=state["starts"], want_lse=True, want_entropy=want)
        return dict(logp=logp, lse=lse, entropy=entropy) if want else dict(logp=logp, lse=lse)
    live, t = _plain_ids(state)
    m, x, e, s = _plain_stats(z)
    log_s = s[:, 0].double().log()                                    # one value a row: 64 bits
    lse = m[:, 0].double() + log_s
    out = dict(logp=torch.where(live, z.gather(1, t)[:, 0].double() - lse, 0.0).float(), lse=torch.where(live, lse, 0.0).float())
    if want:
        out["entropy"] = torch.where(live, log_s - ((e * x).sum(1) / s[:, 0]).double(), 0.0).float()
    return out


CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _policy(state):
    z = state["logits"]
    if own:
        grad, loss, logp, kl, entropy = _ops().policy_grad(
            z, state["ids"], state["advantages"], state["old"], state["valid"], ref_logp=state["ref"], clip=(CLIP_LOW, CLIP_HIGH),
            kl_coef=state["kl_coef"], entropy_coef=state["entropy_coef"], seq_starts=state["starts"], grad=state["grad"])
    else:
        live, t = _plain_ids(state)
        m, x, e, s = _plain_stats(z)
        log_s = s[:, 0].double().log()
        logp = x.gather(1, t)[:, 0].double() - log_s                  # values of one token, in 64 bits
        a = state["advantages"].double()
        rho = torch.exp(logp - state["old"].double())
        clipped = torch.clamp(rho, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
        loss = -torch.minimum(rho * a, clipped * a)
        slope = torch.where(rho * a <= clipped * a, -rho * a, 0.0)
        kl = entropy = None
        if state["ref"] is not None:
            d = state["ref"].double() - logp
            kl = torch.expm1(d) - d
            loss = loss + state["kl_coef"] * kl
            slope = slope - state["kl_coef"] * torch.expm1(d)
        p = e / s
        scale = torch.where(live, 1.0 / state["valid"], 0.0)
        grad = p * (-slope * scale).float()[:, None]
        grad.scatter_add_(1, t, (slope * scale).float()[:, None])
        if state["entropy_coef"]:
            entropy = log_s - (p * x).sum(1).double()
            loss = loss - state["entropy_coef"] * entropy
            grad += p * (x + (entropy - log_s).float()[:, None]) * (state["entropy_coef"] * scale).float()[:, None]
        loss, logp, kl, entropy = (None if v is None else torch.where(live, v, 0.0).float() for v in (loss, logp, kl, entropy))
    out = dict(grad=grad, loss=loss, logp=logp)
    if state["ref"] is not None:
        out["kl"] = kl
    if state["entropy_coef"]:
        out["entropy"] = entropy
    return out


def _preference(state):
    z, case = state["logits"], state["case"]
    if own:
        grad, loss, scores = _ops().preference_grad(z, state["ids"], state["starts"], ref_logp=state["ref"], kind=case["kind"], beta=state["beta"],
                                                    label_smoothing=state["smoothing"], average=case["average"], grad=state["grad"])
        return dict(grad=grad, loss=loss, scores=scores)
    live, t = _plain_ids(state)
    m, x, e, s = _plain_stats(z)
    logp = x.gather(1, t)[:, 0].double() - s[:, 0].double().log()
    starts = state["starts"].long()
    zero = torch.zeros(1, dtype=torch.float64, device=z.device)
    total = torch.cat([zero, torch.where(live, logp - state["ref"].double(), 0.0).cumsum(0)])       # long sums in 64 bits
    count = torch.cat([zero, live.double().cumsum(0)])
    scores, n = total[starts[1:]] - total[starts[:-1]], count[starts[1:]] - count[starts[:-1]]
    n = n.clamp(min=1.0) if case["average"] else torch.ones_like(n)
    scores = scores / n
    delta, beta, eps = scores[0::2] - scores[1::2], state["beta"], state["smoothing"]
    h = beta * delta
    if case["kind"] == "sigmoid":
        soft = torch.log1p(torch.exp(-h.abs()))
        loss = (1.0 - eps) * (soft + (-h).clamp(min=0.0)) + eps * (soft + h.clamp(min=0.0))
        slope = beta * (eps - 1.0 / (1.0 + torch.exp(h)))
    elif case["kind"] == "hinge":
        loss, slope = (1.0 - h).clamp(min=0.0), torch.where(h < 1.0, -beta, 0.0)
    else:
        loss, slope = (delta - 0.5 / beta).square(), 2.0 * (delta - 0.5 / beta)
    slope = torch.stack([slope, -slope], 1).reshape(-1) / n / delta.numel()
    row = torch.repeat_interleave(slope, starts[1:] - starts[:-1], output_size=z.shape[0])
    row = torch.where(live, row, 0.0).float()[:, None]
    grad = (e / s) * -row
    grad.scatter_add_(1, t, row)
    return dict(grad=grad, loss=loss.float(), scores=scores.float())


def _distill(state):
    z, temperature, soft, hard = state["logits"], state["temperature"], state["soft"], state["hard"]
    if own:
        grad, loss = _ops().distill_grad(z, state["teacher_ids"], state["teacher_logits"], state["valid"], temperature=temperature, soft_coef=soft,
                                         hard_coef=hard, targets=state["ids"], weights=state["weights"], seq_starts=state["starts"], grad=state["grad"])
        return dict(grad=grad, loss=loss)
    live, t = _plain_ids(state)
    ids, u = state["teacher_ids"].long(), state["teacher_logits"].float() / temperature
    q = torch.exp(u - u.amax(1, keepdim=True))
    norm = q.sum(1, keepdim=True)
    log_q = (u - u.amax(1, keepdim=True)).double() - norm.double().log()
    q = q / norm
    m = z.amax(1, keepdim=True)
    x = z - m
    e = torch.exp(x / temperature)
    s = e.sum(1, keepdim=True)
    log_p = x.gather(1, ids).double() / temperature - s.double().log()
    weight = torch.where(live, state["weights"], 0.0)
    loss = soft * (q.double() * (log_q - log_p)).sum(1)
    scale = weight[:, None] / state["valid"]
    grad = (e / s) * (scale * (soft / temperature))
    grad.scatter_add_(1, ids, -q * (scale * (soft / temperature)))
    if hard:
        e = torch.exp(x)
        s = e.sum(1, keepdim=True)
        loss = loss - hard * (x.gather(1, t)[:, 0].double() - s[:, 0].double().log())
        grad += (e / s) * (scale * hard)
        grad.scatter_add_(1, t, -scale * hard)
    return dict(grad=grad, loss=(loss * weight.double()).float())


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    rows, vocab = case["rows"], case["vocab"]
    live = sum(_layout(case)[1])
    nbytes = 4 * live * vocab + 4 * rows                              # the supervised rows' logits, the ids
    if case["op"] == "logprobs":
        nbytes += (12 if case["entropy"] else 8) * rows
    else:
        nbytes += 4 * rows * vocab                                    # the gradient, zero rows among it
    if case["op"] == "policy":
        nbytes += 4 * rows * (4 + 2 * case["kl"] + case["entropy"])
    if case["op"] == "preference":
        nbytes += 4 * rows + 6 * case["seqs"]
    if case["op"] == "distill":
        nbytes += rows * case["top_k"] * (8 if case["teacher"] == "float32" else 6) + 8 * rows
    return {"bytes": nbytes, "flops": live * vocab * (4 if case["op"] == "logprobs" else 6)}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    """Losses as functions of the logits by log_softmax, their gradients by differentiation."""
    state = prepare(case, seed)
    logits, rows, vocab = state["logits"], case["rows"], case["vocab"]
    state.pop("grad", None)
    ids = state["ids"].long()
    starts = [0, rows] if state["starts"] is None else state["starts"].tolist()
    keep = (ids >= 0).double()
    safe = ids.clamp(min=0)
    out = {}

    def put(name, part):
        out.setdefault(name, []).append(part.detach())

    upstream = None
    if case["op"] == "preference":                                    # first the pairs' losses as functions of the tokens' log-probabilities
        logp = torch.cat([torch.log_softmax(logits[a:b].double(), 1).gather(1, safe[a:b, None])[:, 0] for a, b in _chunks(rows, vocab, 1 << 26)])
        logp.requires_grad_(True)
        ratio = (logp - state["ref"].double()) * keep
        scores = torch.stack([ratio[a:b].sum() / (keep[a:b].sum().clamp(min=1.0) if case["average"] else 1.0) for a, b in zip(starts, starts[1:])])
        gap = scores[0::2] - scores[1::2]
        h = state["beta"] * gap
        if case["kind"] == "sigmoid":
            e = state["smoothing"]
            loss = -(1.0 - e) * torch.nn.functional.logsigmoid(h) - e * torch.nn.functional.logsigmoid(-h)
        elif case["kind"] == "hinge":
            loss = torch.relu(1.0 - h)
        else:
            loss = (gap - 1.0 / (2.0 * state["beta"])) ** 2
        upstream, = torch.autograd.grad(loss.mean(), logp)
        out = dict(loss=[loss.detach()], scores=[scores.detach()])
    for a, b in _chunks(rows, vocab, 1 << 26):
        z = logits[a:b].double().requires_grad_(True)
        live = keep[a:b]
        lsm = torch.log_softmax(z, 1)
        logp = lsm.gather(1, safe[a:b, None])[:, 0]
        if case["op"] == "logprobs":
            put("logp", logp * live)
            put("lse", torch.logsumexp(z, 1) * live)
            if case["entropy"]:
                put("entropy", -(lsm.exp() * lsm).sum(1) * live)
            continue
        if case["op"] == "preference":
            total = (logp * upstream[a:b]).sum()
        elif case["op"] == "policy":
            ratio = torch.exp(logp - state["old"][a:b].double())
            adv = state["advantages"][a:b].double()
            loss = torch.maximum(-ratio * adv, -ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv)
            if state["ref"] is not None:
                gap = state["ref"][a:b].double() - logp
                kl = torch.exp(gap) - gap - 1.0
                loss = loss + state["kl_coef"] * kl
                put("kl", kl * live)
            if state["entropy_coef"]:
                entropy = -(lsm.exp() * lsm).sum(1)
                loss = loss - state["entropy_coef"] * entropy
                put("entropy", entropy * live)
            put("logp", logp * live)
            put("loss", loss * live)
            total = (loss * live).sum() / state["valid"]
        else:
            t = state["temperature"]
            lq = torch.log_softmax(state["teacher_logits"][a:b].double() / t, 1)
            lp = torch.log_softmax(z / t, 1).gather(1, state["teacher_ids"][a:b].long())
            loss = state["soft"] * torch.nn.functional.kl_div(lp, lq, log_target=True, reduction="none").sum(1) - state["hard"] * logp
            loss = loss * state["weights"][a:b].double() * live
            put("loss", loss)
            total = loss.sum() / state["valid"]
        put("grad", torch.autograd.grad(total, z)[0])
    return {k: torch.cat(v) for k, v in out.items()}
