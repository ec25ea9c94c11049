"""The objectives over logits (seraph_token_logprobs, _policy_grad, _preference_grad, _distill_grad) against their
64-bit definitions, within tolerances that tests/objectives_ref.py derives from the arithmetic."""
import numpy as np
import pytest
import torch

from tests import objectives_ref as ref

pytestmark = pytest.mark.gpu

# one column; fewer columns than a vector; widths around each kernel's limits, multiples of four and not; beyond the
# longest row that fits registers
COLS = [1, 2, 3, 5, 63, 64, 257, 1000, 1023, 1024, 1029, 2048, 4099, 8192, 16385, 32768, 32769, 33001, 50021, 65536, 151936, 151935]


@pytest.fixture(scope="module")
def ops():
    from seraph_amd import ops as o
    o.init(0)
    return o


def dev(a, shift=0):
    """On the device; with a shift, at an address that is 4 shift bytes past a 16-byte boundary."""
    if a is None:
        return None
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    t = torch.from_numpy(a)
    if not shift:
        return t.cuda()
    room = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")
    view = room[shift:].view(t.shape)
    view.copy_(t)
    return view


def check(what, got, want, tol):
    got = got.detach().cpu().numpy().astype(np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want) / tol, 0)), bad.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off; worst at {i}: got {got[i]:.9g} want {want[i]:.9g} tolerance {tol[i]:.3g}")


def make(rows, cols, seed, spread=2.0):
    r = np.random.default_rng(seed)
    z = (spread * r.standard_normal((rows, cols))).astype(np.float32)
    t = r.integers(0, cols, rows).astype(np.uint32)
    return r, z, t


def target_logp(z, t):
    out = np.zeros(len(z))
    for i in range(len(z)):
        if t[i] < z.shape[1]:
            out[i] = ref.log_softmax(z[i:i + 1].astype(np.float64))[0, t[i]]
    return out


def policy_inputs(r, z, t):
    """old policies on both sides of both bounds and well away from them, whatever the logits"""
    logp = target_logp(z, t)
    steps = np.array([0.05, -0.07, 0.6, -0.6, 0.1, -0.45])
    old = (logp - steps[np.arange(len(z)) % 6]).astype(np.float32)
    refl = (logp + 0.3 * r.standard_normal(len(z))).astype(np.float32)
    adv = np.where(np.arange(len(z)) // 6 % 2 == 0, 1.0, -1.0) * (0.5 + r.random(len(z)))
    return adv.astype(np.float32), old, refl


def run_policy(ops, z, t, adv, old, valid, refl=None, weights=None, starts=None, kl=0.0, ent=0.0, shift=0, gshift=None, in_place=False):
    Z = dev(z, shift)
    grad = Z if in_place else None
    if gshift is not None:
        grad = dev(np.full(z.shape, np.nan, np.float32), gshift)
    got = ops.policy_grad(Z, dev(t), dev(adv), dev(old), valid, ref_logp=dev(refl), weights=dev(weights), clip=(0.2, 0.3), kl_coef=kl,
                          entropy_coef=ent, seq_starts=dev(starts), grad=grad, want_entropy=bool(ent))
    torch.cuda.synchronize()
    return dict(zip(("grad", "loss", "logp", "kl", "entropy"), got))


def compare(got, pair, what):
    want, tol = pair
    for k, v in got.items():
        if v is not None:
            check(f"{what} {k}", v, want[k], tol[k])


@pytest.mark.parametrize("cols", COLS)
def test_token_logprobs(ops, cols):
    rows = 5
    r, z, t = make(rows, cols, cols)
    t[1] = cols                                                   # not supervised
    for entropy in (False, True):
        logp, lse, ent = ops.token_logprobs(dev(z), dev(t), want_lse=True, want_entropy=entropy)
        compare(dict(logp=logp, lse=lse, entropy=ent), ref.token_logprobs(z, t), f"{cols}")
    one, none, _ = ops.token_logprobs(dev(z), dev(t))
    assert none is None and torch.equal(one, ops.token_logprobs(dev(z), dev(t), want_lse=True)[0])


@pytest.mark.parametrize("cols", COLS)
def test_policy(ops, cols):
    rows = 13
    r, z, t = make(rows, cols, cols + 1)
    t[3] = 0xffffffff
    adv, old, refl = policy_inputs(r, z, t)
    w = (0.5 + r.random(rows)).astype(np.float32)
    w[4] = 0
    for kw in (dict(), dict(refl=refl, kl=0.05, weights=w), dict(refl=refl, kl=0.05, ent=0.01, weights=w)):
        got = run_policy(ops, z, t, adv, old, rows - 2, **kw)
        want = ref.policy(z, t, adv, old, rows - 2, ref=kw.get("refl"), weights=kw.get("weights"), clip=(0.2, 0.3), kl_coef=kw.get("kl", 0.0),
                          entropy_coef=kw.get("ent", 0.0))
        compare(got, want, f"{cols} {sorted(kw)}")
        again = run_policy(ops, z, t, adv, old, rows - 2, **kw)
        inside = run_policy(ops, z, t, adv, old, rows - 2, in_place=True, **kw)
        for k in got:
            assert got[k] is None or (torch.equal(got[k], again[k]) and torch.equal(got[k], inside[k])), (cols, k)
    zero = run_policy(ops, z, t, adv, old, 0)
    assert (zero["grad"] == 0).all()


@pytest.mark.parametrize("cols", [7, 8192, 33001])
@pytest.mark.parametrize("high", [0.3, float("inf")])
def test_policy_without_advantage_far_from_the_old_policy(ops, cols, high):
    """exp(100) is beyond FP32, not beyond the 64 bits of the definition: 0 times it is 0, and the KL term remains."""
    r, z, t = make(6, cols, cols + 11)
    adv, old, refl = policy_inputs(r, z, t)
    adv[[0, 1, 4]] = [0.0, -0.0, 0.0]
    old[[0, 1]] = (target_logp(z, t)[[0, 1]] - 100.0).astype(np.float32)
    old[5] = np.nan                                               # stays visible in its own row
    adv[5] = 0.0
    g, loss, logp, kl, _ = ops.policy_grad(dev(z), dev(t), dev(adv), dev(old), 6, ref_logp=dev(refl), clip=(0.2, high), kl_coef=0.1)
    want, tol = ref.policy(z, t, adv, old, 6, ref=refl, clip=(0.2, high), kl_coef=0.1)
    cut = lambda d, a: {k: v[:5] for k, v in d.items() if k in a}                  # noqa: E731
    got = dict(grad=g, loss=loss, logp=logp, kl=kl)
    compare(cut(got, got), (cut(want, got), cut(tol, got)), "policy")
    assert torch.isnan(loss[5]) and torch.isnan(g[5]).all() and torch.isfinite(logp).all()


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("hinge", True), ("squared", True)])
def test_preference(ops, cols, kind, average):
    starts = np.array([0, 3, 4, 9, 13, 13, 20], np.uint32)        # ragged; a pair with an empty sequence
    rows = 22                                                     # two rows behind the last sequence
    r, z, t = make(rows, cols, cols + 2)
    t[[0, 5, 16]] = cols
    refl = (target_logp(z, t) + 0.3 * r.standard_normal(rows)).astype(np.float32)
    for kw in (dict(ref=refl), dict(ref=None)):
        want = ref.preference(z, t, starts.astype(int), kind=kind, beta=0.3, eps=0.1, margin=0.2, average=average, **kw)
        res = []
        for in_place in (False, True, False):
            Z = dev(z)
            grad = Z if in_place else dev(np.full(z.shape, np.nan, np.float32))
            g, loss, scores = ops.preference_grad(Z, dev(t), dev(starts), ref_logp=dev(kw["ref"]), kind=kind, beta=0.3, label_smoothing=0.1,
                                                  margin=0.2, average=average, grad=grad)
            res.append((g, loss, scores))
        compare(dict(grad=res[0][0], loss=res[0][1], scores=res[0][2]), want, f"{cols} {kind}")
        for other in res[1:]:
            assert all(torch.equal(a, b) for a, b in zip(res[0], other))


TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def distill_inputs(r, z, top_k, dtype):
    rows, cols = z.shape
    ids = np.stack([r.permutation(cols)[:top_k] if cols >= top_k else r.integers(0, cols, top_k) for _ in range(rows)]).astype(np.uint32)
    teacher = torch.from_numpy((3 * r.standard_normal((rows, top_k))).astype(np.float32)).to(TYPES[dtype])
    return ids, teacher


def run_distill(ops, z, ids, teacher, valid, in_place=False, shift=0, **kw):
    Z = dev(z, shift)
    grad = Z if in_place else dev(np.full(z.shape, np.nan, np.float32), shift)
    for k in ("targets", "teacher_lse", "weights", "seq_starts"):
        if k in kw:
            kw[k] = dev(kw[k])
    g, loss = ops.distill_grad(Z, dev(ids), teacher.cuda(), valid, grad=grad, **kw)
    return dict(grad=g, loss=loss)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("top_k,dtype,temperature,hard", [(1, "float32", 1.0, 0.0), (7, "bfloat16", 2.0, 0.3), (64, "float16", 1.0, 0.3), (300, "float32", 0.5, 0.0),
                                                         (33, "bfloat16", 0.7, 0.3), (20, "float16", 3.0, 0.5)])
def test_distill(ops, cols, top_k, dtype, temperature, hard):
    rows = 6
    r, z, t = make(rows, cols, cols + 3)
    ids, teacher = distill_inputs(r, z, top_k, dtype)             # with few columns: every id many times
    if cols > 8:
        ids[0, 0] = t[0]                                          # the label among the listed
    ids[1, top_k // 2:] = cols + 5                                # a shorter list
    ids[2] = 0xffffffff                                           # no list at all
    t[3] = cols
    w = (0.5 + r.random(rows)).astype(np.float32)
    w[4] = 0
    kw = dict(temperature=temperature, weights=w, targets=t)
    want = ref.distill(z, ids, teacher.float().numpy(), rows - 1, soft=0.7, hard=hard, **kw)
    got = run_distill(ops, z, ids, teacher, rows - 1, soft_coef=0.7, hard_coef=hard, **kw)
    compare(got, want, f"{cols} {top_k}")
    again = run_distill(ops, z, ids, teacher, rows - 1, soft_coef=0.7, hard_coef=hard, **kw)
    inside = run_distill(ops, z, ids, teacher, rows - 1, soft_coef=0.7, hard_coef=hard, in_place=True, **kw)
    for k in got:
        assert torch.equal(got[k], again[k]) and torch.equal(got[k], inside[k]), k


@pytest.mark.parametrize("cols", [9, 8192, 33001, 1300003])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distill_without_its_soft_part(ops, cols, temperature):
    """Nothing of the list counts then, whatever it holds."""
    r, z, t = make(5, cols, cols + 21)
    t[3] = cols
    ids, teacher = distill_inputs(r, z, 5, "float32")
    want = ref.distill(z, ids, teacher.numpy(), 5, soft=0.0, hard=0.8, targets=t, temperature=temperature)
    teacher[1], teacher[2, 2] = float("nan"), float("inf")
    lse = np.array([0.0, np.nan, np.inf, 1.0, -np.inf], np.float32)
    for kw in (dict(), dict(teacher_lse=lse)):
        got = run_distill(ops, z, ids, teacher, 5, soft_coef=0.0, hard_coef=0.8, targets=t, temperature=temperature, **kw)
        compare(got, want, f"{cols}")


@pytest.mark.parametrize("cols", [37, 8192, 40003])
def test_distill_longest_list_and_the_teachers_own_norm(ops, cols):
    rows, top_k = 4, 1024
    r, z, t = make(rows, cols, cols + 4)
    ids = r.integers(0, cols, (rows, top_k)).astype(np.uint32)    # many ids listed twice
    teacher = torch.from_numpy((2 * r.standard_normal((rows, top_k))).astype(np.float32))
    teacher[0, 5:9] = -float("inf")
    teacher[1] = -float("inf")                                    # a list without mass
    lse = (np.log(top_k) + 3 + r.random(rows)).astype(np.float32)
    for kw in (dict(), dict(teacher_lse=lse)):
        want = ref.distill(z, ids, teacher.numpy(), rows, lse=kw.get("teacher_lse"), temperature=1.5)
        compare(run_distill(ops, z, ids, teacher, rows, temperature=1.5, **kw), want, f"{cols} {sorted(kw)}")


@pytest.mark.parametrize("cols", [6, 8192, 8191, 33001, 40000, 1300003])
@pytest.mark.parametrize("shift,gshift", [(1, 1), (2, 3), (3, 0), (0, 2)])
def test_buffers_off_the_16_byte_boundary(ops, cols, shift, gshift):
    rows = 3 if cols < 10 ** 6 else 2
    r, z, t = make(rows, cols, cols + 5)
    adv, old, refl = policy_inputs(r, z, t)
    got = run_policy(ops, z, t, adv, old, rows, refl=refl, kl=0.1, ent=0.02, shift=shift, gshift=gshift)
    compare(got, ref.policy(z, t, adv, old, rows, ref=refl, clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.02), f"{cols}")
    lp, lse, ent = ops.token_logprobs(dev(z, shift), dev(t), want_lse=True, want_entropy=True)
    compare(dict(logp=lp, lse=lse, entropy=ent), ref.token_logprobs(z, t), f"{cols}")
    ids, teacher = distill_inputs(r, z, 5, "float32")
    compare(run_distill(ops, z, ids, teacher, rows, shift=shift), ref.distill(z, ids, teacher.numpy(), rows), f"{cols}")
    starts = np.array([0, 1, rows], np.uint32)
    g, loss, scores = ops.preference_grad(dev(z, shift), dev(t), dev(starts), grad=dev(np.full(z.shape, np.nan, np.float32), gshift))
    compare(dict(grad=g, loss=loss, scores=scores), ref.preference(z, t, starts.astype(int)), f"{cols}")


@pytest.mark.parametrize("cols", [50, 8192, 40001])
def test_rows_that_are_not_supervised_are_not_read(ops, cols):
    """Prompts, the last tokens of sequences, empty sequences and rows behind the last sequence, all full of NaN and infinities."""
    starts = np.array([0, 0, 4, 5, 5, 11, 12], np.uint32)
    rows = 15
    r, z, t = make(rows, cols, cols + 6)
    t[[5, 7]] = cols
    live = ref.supervised(rows, cols, t, None, starts.astype(int))
    assert 0 < live.sum() < rows
    adv, old, refl = policy_inputs(r, z, t)
    for a in (adv, old, refl):
        a[~live] = np.nan
    clean = z.copy()
    z[~live] = np.array([np.nan, np.inf, -np.inf], np.float32)[np.arange(cols) % 3]
    s = starts.astype(int)
    got = run_policy(ops, z, t, adv, old, 4, refl=refl, kl=0.1, ent=0.01, starts=starts, gshift=0)
    compare(got, ref.policy(clean, t, adv, old, 4, ref=refl, clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.01, starts=s), "policy")
    lp, lse, ent = ops.token_logprobs(dev(z), dev(t), seq_starts=dev(starts), want_lse=True, want_entropy=True)
    compare(dict(logp=lp, lse=lse, entropy=ent), ref.token_logprobs(clean, t, s), "logprobs")
    g, loss, scores = ops.preference_grad(dev(z), dev(t), dev(starts), ref_logp=dev(refl), grad=dev(np.full(z.shape, np.nan, np.float32)))
    compare(dict(grad=g, loss=loss, scores=scores), ref.preference(clean, t, s, ref=refl), "preference")
    ids, teacher = distill_inputs(r, clean, 4, "float32")
    inside = ref.supervised(rows, cols, None, None, s)
    z2 = clean.copy()
    z2[~inside] = np.nan
    teacher[~inside] = float("nan")
    compare(run_distill(ops, z2, ids, teacher, 4, seq_starts=starts, hard_coef=0.5, targets=t),
            ref.distill(clean, ids, teacher.numpy(), 4, hard=0.5, targets=t, starts=s), "distill")
    none = np.full(rows, cols, np.uint32)                         # nothing supervised at all
    got = run_policy(ops, z, none, adv, old, 4, refl=refl, kl=0.1, starts=starts, gshift=0)
    assert all((got[k] == 0).all() for k in ("grad", "loss", "logp", "kl"))


@pytest.mark.parametrize("cols", [50, 8192, 40001])
@pytest.mark.parametrize("rows", [11, 400])
def test_rows_ahead_of_the_first_sequence(ops, rows, cols):
    """Offsets that do not start at 0: what lies ahead of the first sequence is not supervised either."""
    starts = np.array([3, 6, rows - 2], np.uint32)
    r, z, t = make(rows, cols, cols + 11)
    live = ref.supervised(rows, cols, t, None, starts.astype(int))
    clean, z2 = z.copy(), z.copy()
    z2[~live] = np.nan
    adv, old, refl = policy_inputs(r, clean, t)
    got = run_policy(ops, z2, t, adv, old, 7, refl=refl, kl=0.1, starts=starts, gshift=0)
    compare(got, ref.policy(clean, t, adv, old, 7, ref=refl, clip=(0.2, 0.3), kl_coef=0.1, starts=starts.astype(int)), "policy")
    for spoil in (0.0, float("nan")):                             # whatever the allocator hands out as scratch
        room = torch.full((rows * 4096,), spoil, device="cuda")
        del room
        g, loss, scores = ops.preference_grad(dev(z2), dev(t), dev(starts), ref_logp=dev(refl))
        compare(dict(grad=g, loss=loss, scores=scores), ref.preference(clean, t, starts.astype(int), ref=refl), "preference")


@pytest.mark.parametrize("batch,cols", [(62, 130), (63, 130), (64, 33001), (65, 130), (300, 33001), (4097, 17)])
def test_many_sequences(ops, batch, cols):
    """More offsets than a wave has lanes, and than it has squared; lengths from 0 to 7."""
    batch += batch % 2
    r = np.random.default_rng(batch)
    starts = np.concatenate([[0], np.cumsum(r.integers(0, 8 if cols < 1000 else 4, batch))]).astype(np.uint32)
    rows = int(starts[-1]) + 3
    r, z, t = make(rows, cols, batch + 1)
    adv, old, refl = policy_inputs(r, z, t)
    s = starts.astype(int)
    got = run_policy(ops, z, t, adv, old, 50, refl=refl, kl=0.1, starts=starts, gshift=0)
    compare(got, ref.policy(z, t, adv, old, 50, ref=refl, clip=(0.2, 0.3), kl_coef=0.1, starts=s), "policy")
    lp, lse, _ = ops.token_logprobs(dev(z), dev(t), seq_starts=dev(starts), want_lse=True)
    compare(dict(logp=lp, lse=lse), ref.token_logprobs(z, t, s), "logprobs")
    g, loss, scores = ops.preference_grad(dev(z), dev(t), dev(starts), ref_logp=dev(refl))
    compare(dict(grad=g, loss=loss, scores=scores), ref.preference(z, t, s, ref=refl), "preference")


def test_offsets_past_32_bits(ops):
    """More logits than 2^31: the last rows of a long call give what a call of their own gives, bit for bit where they lie
    the same way to memory's lines (which lane takes which column follows from that, and from it the order of additions)."""
    rows, cols, last = 66016, 33001, 32
    assert (rows - last) * cols * 4 % 128 == 0
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
    f = torch.empty(rows, device="cuda").normal_(generator=g)
    ids = torch.randint(0, cols, (rows, 6), device="cuda", generator=g, dtype=torch.int32)
    tl = torch.empty(rows, 6, device="cuda").normal_(generator=g)
    t[: rows - last] = torch.where(torch.arange(rows - last, device="cuda") % 64 == 0, t[: rows - last], -1)
    starts = torch.tensor([0, rows - last, rows], dtype=torch.int32, device="cuda")
    part = slice(rows - last, rows)
    zl, tl_, fl, il, ll = (a[part].clone() for a in (z, t, f, ids, tl))
    w = torch.where(t >= 0, 1.0, 0.0)
    want = ops.token_logprobs(zl, tl_, want_lse=True, want_entropy=True)
    got = ops.token_logprobs(z, t, want_lse=True, want_entropy=True)
    # (a call of 32 rows runs them whole, a long one in pieces: equal up to the order of additions)
    for a, b in zip(got, want):
        assert ((a[part] - b).abs() <= 1e-5).all()
    a, b = ops.policy_grad(z, t, f, f, 10, kl_coef=0.1, ref_logp=f), ops.policy_grad(zl, tl_, fl, fl, 10, kl_coef=0.1, ref_logp=fl)
    assert all(x is None or torch.equal(x[part], y) for x, y in zip(a, b))
    del a
    a, b = ops.distill_grad(z, ids, tl, 10, weights=w), ops.distill_grad(zl, il, ll, 10, weights=w[part].clone())
    assert all(torch.equal(x[part], y) for x, y in zip(a, b))
    del a
    ga, la, sa = ops.preference_grad(z, t, starts, ref_logp=f, grad=z)
    p = torch.softmax(zl.double(), 1)
    slope = ga[rows - last, t[rows - last]].double() / (1 - p[0, tl_[0]])                # of the rejected side, from one of its entries
    hot = torch.zeros_like(p).scatter_(1, tl_.long()[:, None], 1.0)
    live = torch.arange(last, device="cuda") < last - 1
    want_g = torch.where(live[:, None], slope * (hot - p), 0.0)
    assert ((ga[part].double() - want_g).abs() <= 1e-4 * want_g.abs() + 1e-9).all() and torch.isfinite(la).all()


def test_pairs_whose_gradient_takes_two_launches(ops):
    """More workgroups than one launch holds.  The slope of the hinge is known, so the definition is a softmax in 64 bits."""
    rows, cols, beta = 8_400_001, 5, 0.25
    g = torch.Generator(device="cuda").manual_seed(9)
    z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, cols + 1, (rows,), device="cuda", generator=g, dtype=torch.int32)
    s = [0, 2_000_000, 4_100_000, 4_100_001, rows - 2]                               # a pair with a side of one token, two rows behind
    starts = torch.tensor(s, dtype=torch.int32, device="cuda")
    got, loss, scores = ops.preference_grad(z, t, starts, kind="hinge", beta=beta, average=True)
    lp = torch.log_softmax(z.double(), 1)
    live = t < cols
    live[[b - 1 for b in s[1:]]] = False
    live[s[-1]:] = False
    hot = torch.zeros_like(lp).scatter_(1, t.long().clamp(max=cols - 1)[:, None], 1.0)
    tl = torch.where(live, (lp * hot).sum(1), 0.0)
    n = [int(live[a:b].sum()) for a, b in zip(s, s[1:])]
    want_scores = torch.stack([tl[a:b].sum() / max(c, 1) for a, b, c in zip(s, s[1:], n)])
    h = beta * (want_scores[0::2] - want_scores[1::2])
    assert (h < 0.9).all()                                                           # both pairs are on the slope
    f = torch.zeros(rows, dtype=torch.float64, device="cuda")
    for q, (a, b, c) in enumerate(zip(s, s[1:], n)):
        f[a:b] = (-beta if q % 2 == 0 else beta) / max(c, 1) / 2
    f = torch.where(live, f, 0.0)[:, None]
    p = lp.exp()
    spread = (z.max(1).values - z.min(1).values).double()
    u = ref.HALF_STEP * (6.0 * spread + cols / 64.0 + 40.0)                          # ref.unit
    assert ((got.double() - f * (hot - p)).abs() <= f.abs() * 2 * u[:, None] * (p + hot) + 1e-38).all()
    err = float(u.max())
    assert ((scores.double() - want_scores).abs() <= err + ref.HALF_STEP * want_scores.abs()).all()
    assert ((loss.double() - (1.0 - h)).abs() <= 2 * beta * err + ref.HALF_STEP * (1.0 - h).abs()).all()


@pytest.mark.parametrize("cols", [9, 1000, 8192, 33000, 151936])
def test_masked_logits_inside_a_row(ops, cols):
    """Entries of -inf and of the type's lowest value, rows where a single entry is left, rows of nothing but lowest values,
    and values far from zero."""
    rows = 12
    r, z, t = make(rows, cols, cols + 7)
    low = np.finfo(np.float32).min
    t[:] = r.integers(0, 4, rows)
    z[0, 4:] = -np.inf
    z[1, 4:] = low
    z[2] = -np.inf; z[2, t[2]] = 3.0
    z[3] = low; z[3, t[3]] = 1.0
    z[4] = low                                                    # uniform
    z[5] += 1e4
    z[6] -= 1e4
    z[7, ::2] = -np.inf; z[7, t[7]] = 0.5
    z[8] = 0.0
    z[9, cols // 2] = 300.0
    z[10, :] = -np.inf; z[10, t[10]] = low
    z[11, 4:] = -1e30
    adv, old, refl = policy_inputs(r, z, t)
    got = run_policy(ops, z, t, adv, old, rows, refl=refl, kl=0.1, ent=0.01)
    compare(got, ref.policy(z, t, adv, old, rows, ref=refl, clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.01), "policy")
    lp, lse, ent = ops.token_logprobs(dev(z), dev(t), want_lse=True, want_entropy=True)
    compare(dict(logp=lp, lse=lse, entropy=ent), ref.token_logprobs(z, t), "logprobs")
    starts = np.array([0, 6, 12], np.uint32)
    g, loss, scores = ops.preference_grad(dev(z), dev(t), dev(starts), ref_logp=dev(refl))
    compare(dict(grad=g, loss=loss, scores=scores), ref.preference(z, t, starts.astype(int), ref=refl), "preference")
    ids = np.tile(np.arange(4, dtype=np.uint32), (rows, 1))
    teacher = torch.from_numpy(r.standard_normal((rows, 4)).astype(np.float32))
    teacher[(2, 3, 7, 10), :] = -float("inf")                     # mass only where the student can follow
    for i in (2, 3, 7, 10):
        teacher[i, int(t[i])] = 1.0
    for temperature, hard in ((1.0, 0.0), (2.0, 0.5), (1.7, 0.5)):
        want = ref.distill(z, ids, teacher.numpy(), rows, temperature=temperature, hard=hard, targets=t)
        compare(run_distill(ops, z, ids, teacher, rows, temperature=temperature, hard_coef=hard, targets=t), want, f"distill {temperature}")


@pytest.mark.parametrize("cols", [100, 8192, 40000])
def test_nan_and_inf_stay_in_their_row(ops, cols):
    r, z, t = make(6, cols, cols + 8)
    z[1, 3] = np.nan
    z[3, 5] = np.inf
    z[4] = -np.inf
    adv, old, refl = policy_inputs(r, z, t)
    old[:], refl[:] = -5.0, -5.0
    got = run_policy(ops, z, t, adv, old, 6, refl=refl, kl=0.1, ent=0.01)
    for i in range(6):
        assert torch.isnan(got["grad"][i]).all().item() == (i in (1, 3, 4)) and torch.isnan(got["logp"][i]).item() == (i in (1, 3, 4)), i
        assert torch.isfinite(got["grad"][i]).all().item() == (i not in (1, 3, 4))
    ids, teacher = distill_inputs(r, z, 3, "float32")
    teacher[0, 1] = float("nan")
    got = run_distill(ops, z, ids, teacher, 6)
    for i in range(6):
        assert torch.isnan(got["grad"][i]).all().item() == (i in (0, 1, 3, 4)), i


@pytest.mark.parametrize("rows,cols", [(3000, 1029), (1, 151936), (700, 33000), (300, 65537)])
def test_many_rows_and_one(ops, rows, cols):
    """More rows than workgroups that fit the chip, and a single one; checked on the device in 64 bits by torch."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
    lsm = torch.log_softmax(z.double(), 1)
    want = lsm.gather(1, t.long()[:, None])[:, 0]
    u = float(ref.unit(z[:1].cpu().numpy())[0, 0]) * 2            # the rows are alike; twice one row's bound
    logp, _, ent = ops.token_logprobs(z, t, want_entropy=True)
    assert ((logp.double() - want).abs() <= u + ref.HALF_STEP * want.abs()).all()
    old = (want - 0.1).float()
    adv = torch.ones(rows, device="cuda")
    grad, loss, lp, _, _ = ops.policy_grad(z, t, adv, old, rows, weights=torch.full((rows,), 2.0, device="cuda"))
    rho = torch.exp(want - old.double())
    p = lsm.exp()
    hot = torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0)
    f = (2.0 / rows) * rho[:, None]
    assert ((grad.double() - f * (p - hot)).abs() <= 4 * u * f * (p + hot)).all()
    assert ((lp.double() - want).abs() <= u + ref.HALF_STEP * want.abs()).all()
    k = 5
    ids = torch.stack([torch.randperm(cols, device="cuda", generator=g)[:k] for _ in range(rows)]).to(torch.int32)
    tl = torch.empty(rows, k, device="cuda").normal_(generator=g)
    q = torch.softmax(tl.double(), 1)
    grad, loss = ops.distill_grad(z, ids, tl, rows)
    want_g = p.scatter_add(1, ids.long(), -q) / rows
    assert ((grad.double() - want_g).abs() <= 4 * u * (p + torch.zeros_like(p).scatter_(1, ids.long(), q)) / rows).all()
    wl = (q * (q.log() - lsm.gather(1, ids.long()))).sum(1)
    assert ((loss.double() - wl).abs() <= 4 * u * (1 + wl.abs() + q.log().abs().max())).all()


@pytest.mark.parametrize("cols", [13, 8192, 40001])
def test_gradients_against_differences(ops, cols):
    """The gradient of each op against central differences of the op's own loss, at entries that carry it.  With a step
    of h = 1/16 the difference is off by h^2 |f'''| / 6, |f'''| at most the row's factor times 8, plus the loss's own
    error (the bound of the 64-bit definition) over h."""
    rows, h = 4, 1.0 / 16
    r, z, t = make(rows, cols, cols + 9, spread=0.5)
    z[np.arange(rows), t] += np.log(cols)                         # probabilities that differences can see
    adv, old, refl = policy_inputs(r, z, t)
    old = (target_logp(z, t) - 0.05).astype(np.float32)           # inside the bounds for every step
    starts = np.array([0, 2, 4], np.uint32)
    ids, teacher = distill_inputs(r, z, 3, "float32")
    ids[:, 0] = t

    def policy(x):
        return run_policy(ops, x, t, adv, old, 1, refl=refl, kl=0.1, ent=0.01)

    def pref(x):
        g, loss, _ = ops.preference_grad(dev(x), dev(t), dev(starts), ref_logp=dev(refl), beta=0.5)
        return dict(grad=g, loss=loss)

    def dist(x):
        return run_distill(ops, x, ids, teacher, 1, temperature=1.5, hard_coef=0.4, targets=t)
    lt = {policy: ref.policy(z, t, adv, old, 1, ref=refl, clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.01)[1]["loss"].sum(),
          pref: ref.preference(z, t, starts.astype(int), ref=refl, beta=0.5)[1]["loss"].sum(),
          dist: ref.distill(z, ids, teacher.numpy(), 1, temperature=1.5, hard=0.4, targets=t)[1]["loss"].sum()}
    for f in (policy, pref, dist):
        grad = f(z)["grad"].cpu().numpy().astype(np.float64)
        for row in range(rows):
            for c in (int(t[row]), int(ids[row, 1]), (int(t[row]) + 1) % cols):
                a, b = z.copy(), z.copy()
                a[row, c] += h
                b[row, c] -= h
                step = float(a[row, c]) - float(b[row, c])
                d = (f(a)["loss"].double().sum() - f(b)["loss"].double().sum()).item() / step
                if f is pref:
                    d /= 1                                        # one pair: the mean is the loss
                assert abs(d - grad[row, c]) <= h * h * 8 * 2.0 / 6 + 2 * 2 * lt[f] / step, (f.__name__, row, c, d, grad[row, c])


def test_captured_and_replayed(ops):
    """Each op captured into a graph, replayed on new inputs with eager work in between, against the eager result."""
    for rows, cols in ((7, 8191), (9, 40000)):
        r, z, t = make(rows, cols, cols)
        adv, old, refl = policy_inputs(r, z, t)
        ids, teacher = distill_inputs(r, z, 8, "float32")
        starts = np.array([0, 3, rows], np.uint32)
        Z, T, A, O, R, I, L, S = (dev(a) for a in (z, t, adv, old, refl, ids, teacher.numpy(), starts))
        calls = (lambda: ops.policy_grad(Z, T, A, O, rows, ref_logp=R, kl_coef=0.1, entropy_coef=0.01),
                 lambda: ops.preference_grad(Z, T, S, ref_logp=R), lambda: ops.distill_grad(Z, I, L, rows, targets=T, hard_coef=0.5, temperature=2.0),
                 lambda: ops.token_logprobs(Z, T, want_lse=True, want_entropy=True))
        for call in calls:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call()
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = call()
            for k in range(4):
                Z.copy_(dev((2 * np.random.default_rng(100 + k).standard_normal((rows, cols))).astype(np.float32)))
                want = call()
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                for a, b in zip(out, want):
                    assert a is None or torch.equal(a, b)


def test_two_streams_at_once(ops):
    """Calls on two streams over long rows, started together, give what each gives alone."""
    rows, cols = 600, 40001
    data = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
        t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
        lp, _, _ = ops.token_logprobs(z, t)
        data.append((z, t, lp, torch.ones(rows, device="cuda")))
    alone = [ops.policy_grad(z, t, a, lp, rows) for z, t, lp, a in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = []
    for _ in range(3):
        for s, (z, t, lp, a) in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(ops.policy_grad(z, t, a, lp, rows))
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        assert all(x is None or torch.equal(x, y) for x, y in zip(res, alone[i % 2]))


@pytest.mark.parametrize("rows,cols", [(5, 40001), (700, 65536), (3, 1200000)])
@pytest.mark.parametrize("spins", [0, 1])
def test_long_rows_when_partners_are_not_waited_for(ops, rows, cols, spins):
    """Whoever learns a part's statistics in whichever way, the bits are the same; in place too."""
    from seraph_amd._lib import kernels
    g = torch.Generator(device="cuda").manual_seed(rows)
    z = torch.empty(rows, cols, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[1] = -1
    old, adv = torch.full((rows,), -11.0, device="cuda"), torch.ones(rows, device="cuda")
    ids = torch.randint(0, cols + 9, (rows, 33), device="cuda", generator=g, dtype=torch.int32)
    tl = torch.empty(rows, 33, device="cuda").normal_(generator=g)
    calls = [lambda x, out: ops.policy_grad(x, t, adv, old, rows, ref_logp=old, kl_coef=0.1, grad=out),
             lambda x, out: ops.policy_grad(x, t, adv, old, rows, entropy_coef=0.1, grad=out),
             lambda x, out: ops.distill_grad(x, ids, tl, rows, grad=out),
             lambda x, out: ops.distill_grad(x, ids, tl, rows, temperature=2.0, hard_coef=0.5, targets=t, grad=out),
             lambda x, out: ops.distill_grad(x, ids, tl, rows, temperature=1.5, hard_coef=0.5, targets=t, grad=out)]
    for call in calls:
        want = call(z, None)
        try:
            kernels().seraph_objectives_exchange_spins(spins)
            for x in (z, z.clone()):
                got = call(x, None if x is z else x)
                torch.cuda.synchronize()
                assert all(a is None or torch.equal(a, b) for a, b in zip(got, want))
        finally:
            kernels().seraph_objectives_exchange_spins(1 << 16)


def test_wrapper_refusals(ops):
    from seraph_amd._lib import SeraphError
    z, t, f = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    s = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.token_logprobs(z.half(), t), lambda: ops.token_logprobs(z.t(), t), lambda: ops.token_logprobs(z, t.long()),
                lambda: ops.token_logprobs(z, t[:3]), lambda: ops.token_logprobs(z, t.cpu()), lambda: ops.token_logprobs(z[:, :0], t),
                lambda: ops.policy_grad(z, t, f, f[:3], 4), lambda: ops.policy_grad(z, t, f, f, 4, kl_coef=0.1),
                lambda: ops.policy_grad(z, t, f, f, 4, grad=z[:2]), lambda: ops.policy_grad(z, t, f, f, 4, clip=(-1.0, 0.2)),
                lambda: ops.preference_grad(z, t, s[:2]), lambda: ops.preference_grad(z, t, None), lambda: ops.preference_grad(z, t, s, kind="x"),
                lambda: ops.preference_grad(z, t, s, beta=0.0), lambda: ops.distill_grad(z, t, f, 4),
                lambda: ops.distill_grad(z, t[:, None], f[:, None].double(), 4), lambda: ops.distill_grad(z, t[:, None], f[:, None], 4, hard_coef=1.0),
                lambda: ops.distill_grad(z, t[:, None], f[:, None], 4, temperature=0.0),
                lambda: ops.distill_grad(z, torch.zeros(4, 1025, dtype=torch.int32, device="cuda"), torch.zeros(4, 1025, device="cuda"), 4)):
        with pytest.raises(SeraphError):
            bad()
    empty = torch.zeros(0, 8, device="cuda")
    lp, _, _ = ops.token_logprobs(empty, t[:0])
    assert lp.numel() == 0
