"""The 64-bit definitions that the objectives are tested against: their gradients against central differences of their
own losses, and the refusals of the C interface, none of which needs a device."""
import ctypes as C
import os

import numpy as np
import pytest

from tests import objectives_ref as ref


def numeric(f, z, eps=1e-5):
    g = np.zeros(z.shape)
    for i in np.ndindex(z.shape):
        a, b = z.copy(), z.copy()
        a[i] += eps
        b[i] -= eps
        g[i] = (f(a) - f(b)) / (2 * eps)
    return g


def close(got, want):
    # eps^2 f'''/6 + 2^-53 |f| / eps with eps = 1e-5, |f'''| < 20 and |f| < 100
    assert np.abs(got - want).max() <= 1e-10 * 20 / 6 + 100 * 2.0 ** -52 / 1e-5


def inputs(seed, rows, cols):
    r = np.random.default_rng(seed)
    z = r.standard_normal((rows, cols))
    return r, z, r.integers(0, cols, rows)


@pytest.mark.parametrize("kl,ent", [(0.0, 0.0), (0.3, 0.0), (0.2, 0.1)])
def test_policy_gradient_is_its_losses_derivative(kl, ent):
    r, z, a = inputs(1, 6, 5)
    logp = np.array([ref.log_softmax(z[i:i + 1])[0, a[i]] for i in range(6)])
    old, refl = logp + np.array([0.05, -0.05, 0.5, -0.5, 0.5, -0.5]), logp + 0.3 * r.standard_normal(6)
    adv = np.array([1.0, -1.0, 1.0, 1.0, -1.0, -1.0])                       # both sides of both bounds
    w = np.array([1.0, 0.5, 2.0, 1.0, 1.0, 0.0])
    kw = dict(ref=refl, weights=w, clip=(0.2, 0.3), kl_coef=kl, entropy_coef=ent)
    out, _ = ref.policy(z, a, adv, old, 5, **kw)
    close(out["grad"], numeric(lambda x: ref.policy(x, a, adv, old, 5, **kw)[0]["loss"].sum() / 5, z))


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("average", [False, True])
def test_preference_gradient_is_its_losses_derivative(kind, average):
    r, z, t = inputs(2, 11, 4)
    starts = [0, 3, 7, 9, 11]
    kw = dict(ref=r.standard_normal(11) - 1, kind=kind, beta=0.5, eps=0.1, margin=0.2, average=average)
    out, _ = ref.preference(z, t, starts, **kw)
    close(out["grad"], numeric(lambda x: ref.preference(x, t, starts, **kw)[0]["loss"].mean(), z))


@pytest.mark.parametrize("temperature,hard,own_lse", [(1.0, 0.0, False), (2.0, 0.4, False), (0.5, 0.4, True)])
def test_distill_gradient_is_its_losses_derivative(temperature, hard, own_lse):
    r, z, t = inputs(3, 5, 7)
    ids = np.array([[0, 3, 6], [1, 1, 2], [5, 9, 0], [4, 3, 2], [6, 6, 6]])  # ids listed twice, an id past the end
    teacher = r.standard_normal((5, 3)).astype(np.float32)
    kw = dict(temperature=temperature, soft=0.7, hard=hard, targets=t, lse=np.full(5, 2.0) if own_lse else None, weights=np.array([1, 2, 0.5, 1, 0]))
    out, _ = ref.distill(z, ids, teacher, 4, **kw)
    close(out["grad"], numeric(lambda x: ref.distill(x, ids, teacher, 4, **kw)[0]["loss"].sum() / 4, z))


# ------------------------------------------------------------------ refusals, before anything is launched
@pytest.fixture(scope="module")
def k():
    from seraph_amd import _lib
    if not os.path.exists(_lib.KERNEL_LIB):
        from seraph_amd import build
        build.build_all()
    return _lib.kernels()


P = 4096                                                                    # an address that no refused call touches


def refused(k, rc, code, word):
    assert rc == code and word.encode() in k.seraph_hip_last_error(), (rc, k.seraph_hip_last_error())


def test_token_logprobs_refusals(k):
    f = lambda logits=P, t=P, out=P, starts=None, batch=1, rows=4, cols=8: k.seraph_token_logprobs(      # noqa: E731
        logits, t, out, None, None, starts, batch, rows, cols, None, 0, None)
    assert f(rows=0) == 0 and f(cols=0) == 0 and f(logits=None, rows=0) == 0
    refused(k, f(logits=None), -1, "NULL")
    refused(k, f(t=None), -1, "NULL")
    refused(k, f(out=None), -1, "NULL")
    refused(k, f(rows=-1), -1, "shape")
    refused(k, f(cols=1 << 31), -1, "shape")
    refused(k, f(starts=P, batch=0), -1, "batch")


def test_policy_refusals(k):
    from seraph_amd._lib import PolicyOptions

    def f(logits=P, old=P, refl=P, kl_rows=None, o=(0.2, 0.2, 0.1, 0.0), rows=4, cols=8, starts=None, batch=1, ws=None, n=0):
        opt = PolicyOptions(*o) if o else None
        return k.seraph_policy_grad(logits, P, P, old, refl, None, P, P, None, kl_rows, None, opt, starts, batch, rows, cols, 4, ws, n, None)
    assert f(rows=0) == 0 and f(cols=0) == 0
    refused(k, f(logits=None), -1, "NULL")
    refused(k, f(old=None), -1, "NULL")
    refused(k, f(o=None), -1, "NULL")
    refused(k, f(refl=None), -1, "ref_logp")
    refused(k, f(refl=None, o=(0.2, 0.2, 0.0, 0.0), kl_rows=P), -1, "ref_logp")
    refused(k, f(o=(-0.1, 0.2, 0.0, 0.0)), -1, "clip")
    refused(k, f(o=(0.1, float("nan"), 0.0, 0.0)), -1, "clip")
    refused(k, f(o=(0.1, 0.1, float("inf"), 0.0)), -1, "finite")
    refused(k, f(starts=P, batch=0), -1, "batch")
    refused(k, f(rows=1 << 31), -1, "shape")


def test_preference_refusals(k):
    from seraph_amd._lib import PreferenceOptions
    need = k.seraph_preference_grad_ws_bytes(4, 8)
    assert need > 0 and k.seraph_preference_grad_ws_bytes(0, 8) == 0

    def f(logits=P, o=(0, 0.1, 0.0, 0.0, 0), starts=P, pairs=1, rows=4, cols=8, ws=P, n=need):
        opt = PreferenceOptions(*o) if o else None
        return k.seraph_preference_grad(logits, P, None, P, P, None, None, opt, starts, pairs, rows, cols, ws, n, None)
    assert f(rows=0) == 0
    refused(k, f(logits=None), -1, "NULL")
    refused(k, f(o=None), -1, "NULL")
    refused(k, f(starts=None), -1, "NULL")
    refused(k, f(pairs=0), -1, "pairs")
    refused(k, f(o=(3, 0.1, 0.0, 0.0, 0)), -1, "unknown")
    refused(k, f(o=(0, 0.0, 0.0, 0.0, 0)), -1, "beta")
    refused(k, f(o=(0, float("inf"), 0.0, 0.0, 0)), -1, "beta")
    refused(k, f(o=(0, 0.1, 1.5, 0.0, 0)), -1, "smoothing")
    refused(k, f(o=(0, 0.1, 0.0, float("nan"), 0)), -1, "margin")
    refused(k, f(ws=None), -3, "scratch")
    refused(k, f(n=need - 1), -3, "scratch")
    refused(k, f(ws=P + 4), -3, "aligned")


def test_distill_refusals(k):
    from seraph_amd._lib import DistillOptions

    def f(ids=P, targets=None, o=(1.0, 1.0, 0.0, 0), rows=4, cols=8, top_k=2, starts=None, batch=1):
        opt = DistillOptions(*o) if o else None
        return k.seraph_distill_grad(P, ids, P, None, targets, None, P, P, opt, starts, batch, rows, cols, top_k, 4, None, 0, None)
    assert f(rows=0) == 0 and f(cols=0) == 0
    refused(k, f(ids=None), -1, "NULL")
    refused(k, f(o=None), -1, "NULL")
    refused(k, f(top_k=0), -1, "top_k")
    refused(k, f(top_k=1025), -1, "top_k")
    refused(k, f(o=(0.0, 1.0, 0.0, 0)), -1, "temperature")
    refused(k, f(o=(float("nan"), 1.0, 0.0, 0)), -1, "temperature")
    refused(k, f(o=(1.0, float("inf"), 0.0, 0)), -1, "finite")
    refused(k, f(o=(1.0, 1.0, 0.0, 3)), -1, "type")
    refused(k, f(o=(1.0, 1.0, 0.5, 0)), -1, "targets")
    refused(k, f(starts=P, batch=0), -1, "batch")


def test_wrappers_refuse_what_is_not_on_the_device():
    import torch

    from seraph_amd import ops
    from seraph_amd._lib import SeraphError
    z = torch.zeros(4, 8)
    ids = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.token_logprobs(z, ids), lambda: ops.policy_grad(z, ids, z[:, 0], z[:, 0], 4),
                 lambda: ops.preference_grad(z, ids, ids), lambda: ops.distill_grad(z, ids, z, 4)):
        with pytest.raises(SeraphError, match="CUDA"):
            call()


def test_more_rows_than_a_launch_holds(k):
    from seraph_amd._lib import DistillOptions, PolicyOptions, PreferenceOptions
    rows = 1 << 24
    refused(k, k.seraph_token_logprobs(P, P, P, None, None, None, 1, rows, 8, None, 0, None), -1, "shape")
    refused(k, k.seraph_policy_grad(P, P, P, P, None, None, P, P, None, None, None, PolicyOptions(0.2, 0.2, 0.0, 0.0), None, 1, rows, 8, 4, None, 0, None), -1, "shape")
    refused(k, k.seraph_distill_grad(P, P, P, None, None, None, P, P, DistillOptions(1.0, 1.0, 0.0, 0), None, 1, rows, 8, 2, 4, None, 0, None), -1, "shape")
    o = PreferenceOptions(0, 0.1, 0.0, 0.0, 0)
    refused(k, k.seraph_preference_grad(P, P, None, P, P, None, None, o, P, 1, rows, 8, P, 1 << 60, None), -1, "shape")
    refused(k, k.seraph_preference_grad(P, P, None, P, P, None, None, o, P, 1 << 22, 4, 8, P, 1 << 60, None), -1, "pairs")


@pytest.mark.parametrize("off", [4, -4, 4 * 31, -4 * 31])
def test_a_gradient_over_other_logits_than_its_own(k, off):
    from seraph_amd._lib import DistillOptions, PolicyOptions, PreferenceOptions
    g = P + off                                                                          # 4 x 8 logits: 128 bytes
    refused(k, k.seraph_policy_grad(P, P, P, P, None, None, g, P, None, None, None, PolicyOptions(0.2, 0.2, 0.0, 0.0), None, 1, 4, 8, 4, None, 0, None), -1, "overlap")
    refused(k, k.seraph_distill_grad(P, P, P, None, None, None, g, P, DistillOptions(1.0, 1.0, 0.0, 0), None, 1, 4, 8, 2, 4, None, 0, None), -1, "overlap")
    refused(k, k.seraph_preference_grad(P, P, None, g, P, None, None, PreferenceOptions(0, 0.1, 0.0, 0.0, 0), P, 1, 4, 8, P, 1 << 60, None), -1, "overlap")
