"""The objectives over logits from their definitions, in 64 bits (numpy), with bounds on the error that FP32 kernels may
make: every function returns values and, beside them, tolerances that follow from the arithmetic.

A kernel forms e_j = 2^((z_j - m) k) and s = sum e_j in FP32 and everything that is one value a row in 64 bits.
With u = 2^-24 (half a step of FP32) the argument of the exponential has the relative error 3u (a rounded difference,
the rounded constant k, a rounded product), hence e_j the relative error u (3 D / T + 2) with D = max |z - m| over the
entries that are not negligible and one step (2u) for the exponential itself.  s adds at most (n / 64 + 24) u for
additions (64 lanes or more each add at most n / 64 values one after another, then a tree), and the products with
row factors a few u more.  U below is the sum of these, doubled where two such errors meet."""
import numpy as np

HALF_STEP = 2.0 ** -24


def unit(z, inv_temp=1.0):
    """[rows, 1]: relative error of a probability and absolute error of a log-probability of the row."""
    z = np.asarray(z, np.float64)
    finite = np.isfinite(z)
    m = np.max(np.where(finite, z, -np.inf), axis=1, keepdims=True)
    d = np.where(finite, m - z, 0.0)
    d = np.where(d * inv_temp > 110.0, 0.0, d)          # below 2^-149 of the maximum: exactly 0 in both
    D = d.max(axis=1, keepdims=True) * inv_temp
    return HALF_STEP * (6.0 * D + z.shape[1] / 64.0 + 40.0)


def log_softmax(z):
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = z - z.max(axis=1, keepdims=True)
        return x - np.log(np.exp(x).sum(axis=1, keepdims=True))


def supervised(rows, cols, targets=None, weights=None, starts=None):
    live = np.ones(rows, bool)
    if targets is not None:
        live &= targets < cols
    if weights is not None:
        live &= weights != 0
    if starts is not None:
        inside = np.zeros(rows, bool)
        for a, b in zip(starts[:-1], starts[1:]):
            if b > a:
                inside[a:b - 1] = True
        live &= inside
    return live


def _xlogx(p, lp):
    return np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0)


def token_logprobs(z, targets, starts=None):
    rows, cols = z.shape
    live = supervised(rows, cols, targets, None, starts)
    out = {k: np.zeros(rows) for k in ("logp", "lse", "entropy")}
    tol = {k: np.zeros(rows) for k in out}
    for r in np.flatnonzero(live):
        x = z[r:r + 1].astype(np.float64)
        lp = log_softmax(x)[0]
        u = unit(x)[0, 0]
        p = np.exp(lp)
        fin = p > 0
        spread = float((p[fin] * (x.max() - x[0][fin])).sum())
        out["logp"][r] = lp[targets[r]]
        out["lse"][r] = x.max() - lp.max()
        out["entropy"][r] = -_xlogx(p, lp).sum()
        tol["logp"][r] = u + HALF_STEP * abs(lp[targets[r]]) if np.isfinite(lp[targets[r]]) else 0.0
        tol["lse"][r] = u + HALF_STEP * abs(out["lse"][r])
        tol["entropy"][r] = 2 * u * (1.0 + spread) + HALF_STEP * abs(out["entropy"][r])
    return out, tol


def policy(z, actions, adv, old, valid, ref=None, weights=None, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0, starts=None):
    rows, cols = z.shape
    live = supervised(rows, cols, actions, weights, starts)
    scale = 1.0 / valid if valid > 0 else 0.0
    out = {k: np.zeros(rows) for k in ("loss", "logp", "kl", "entropy")}
    tol = {k: np.zeros(rows) for k in out}
    grad, tgrad = np.zeros(z.shape), np.zeros(z.shape)
    for r in np.flatnonzero(live):
        x = z[r:r + 1].astype(np.float64)
        lp = log_softmax(x)[0]
        p = np.exp(lp)
        u = unit(x)[0, 0]
        w = float(weights[r]) if weights is not None else 1.0
        A = float(adv[r])
        logp = lp[actions[r]]
        rho = np.exp(logp - float(old[r]))
        free, held = rho * A, np.clip(rho, 1.0 - float(np.float32(clip[0])), 1.0 + float(np.float32(clip[1]))) * A
        loss, slope, size = -min(free, held), (-free if free <= held else 0.0), abs(free)
        kl_c, ent_c = float(np.float32(kl_coef)), float(np.float32(entropy_coef))
        if ref is not None:
            d = float(ref[r]) - logp
            kl = np.expm1(d) - d
            out["kl"][r] = kl
            tol["kl"][r] = abs(np.expm1(d)) * u + u * u + HALF_STEP * kl
            loss += kl_c * kl
            slope += kl_c * (1.0 - np.exp(d))
            size += abs(kl_c) * np.exp(d)
        H = -_xlogx(p, lp).sum()
        fin = p > 0
        spread = float((p[fin] * (x.max() - x[0][fin])).sum())
        onehot = np.zeros(cols)
        onehot[actions[r]] = 1.0
        g = slope * (onehot - p)
        t = 2 * u * (size + abs(slope)) * (p + onehot)
        if entropy_coef:
            g = g + ent_c * (_xlogx(p, lp) + p * H)
            t = t + 2 * u * abs(ent_c) * p * (np.abs(np.where(fin, lp, 0.0)) + 2 * H + 2 * spread + 2.0)
            loss -= ent_c * H
        out["entropy"][r], tol["entropy"][r] = H, 2 * u * (1.0 + spread) + HALF_STEP * abs(H)
        out["logp"][r], tol["logp"][r] = logp, u + HALF_STEP * abs(logp)
        out["loss"][r] = w * loss
        tol["loss"][r] = abs(w) * (2 * u * size + abs(kl_c) * tol["kl"][r] + abs(ent_c) * tol["entropy"][r] + HALF_STEP * abs(loss))
        grad[r], tgrad[r] = g * w * scale, t * abs(w) * scale
    out["grad"], tol["grad"] = grad, tgrad + 1e-38
    return out, tol


def preference(z, targets, starts, ref=None, kind="sigmoid", beta=0.1, eps=0.0, margin=0.0, average=False):
    rows, cols = z.shape
    beta, eps, margin = (float(np.float32(v)) for v in (beta, eps, margin))
    live = supervised(rows, cols, targets, None, starts)
    lp = np.zeros(rows)
    u = np.zeros(rows)
    for r in np.flatnonzero(live):
        x = z[r:r + 1].astype(np.float64)
        lp[r], u[r] = log_softmax(x)[0][targets[r]], unit(x)[0, 0]
    batch = len(starts) - 1
    score, n, err = np.zeros(batch), np.ones(batch), np.zeros(batch)
    for q in range(batch):
        idx = np.flatnonzero(live[starts[q]:starts[q + 1]]) + starts[q]
        if average and len(idx):
            n[q] = len(idx)
        score[q] = (lp[idx] - (ref[idx].astype(np.float64) if ref is not None else 0.0)).sum() / n[q]
        err[q] = u[idx].sum() / n[q]
    gap, gerr = score[0::2] - score[1::2], err[0::2] + err[1::2]
    h = beta * gap - margin
    sig = 1.0 / (1.0 + np.exp(-h))
    if kind == "sigmoid":
        loss = (1 - eps) * np.logaddexp(0, -h) + eps * np.logaddexp(0, h)
        slope, serr, lerr = beta * (eps - (1 - sig)), beta * beta * gerr / 4, beta * gerr
    elif kind == "hinge":
        loss, slope = np.maximum(0, 1 - h), np.where(h < 1, -beta, 0.0)
        serr, lerr = 0 * gerr, beta * gerr
    else:
        d = gap - 0.5 / beta
        loss, slope, serr, lerr = d * d, 2 * d, 2 * gerr, 2 * np.abs(d) * gerr + gerr ** 2
    out = dict(loss=loss, scores=score)
    tol = dict(loss=lerr + HALF_STEP * np.abs(loss) + 1e-38, scores=err + HALF_STEP * np.abs(score))
    grad, tgrad = np.zeros(z.shape), np.zeros(z.shape)
    for q in range(batch):
        f = (slope if q % 2 == 0 else -slope)[q // 2] / n[q] / (batch // 2)
        fe = serr[q // 2] / n[q] / (batch // 2)
        for r in range(starts[q], starts[q + 1]):
            if live[r]:
                p = np.exp(log_softmax(z[r:r + 1].astype(np.float64))[0])
                onehot = np.zeros(cols)
                onehot[targets[r]] = 1.0
                grad[r] = f * (onehot - p)
                tgrad[r] = (abs(f) * 2 * u[r] + fe) * (p + onehot)
    out["grad"], tol["grad"] = grad, tgrad + 1e-38
    return out, tol


def distill(z, ids, teacher, valid, temperature=1.0, soft=1.0, hard=0.0, targets=None, lse=None, weights=None, starts=None):
    """teacher: the listed logits as FP32 (their own type is exact in it)."""
    rows, cols = z.shape
    live = supervised(rows, cols, None, weights, starts)
    scale = 1.0 / valid if valid > 0 else 0.0
    soft, hard = float(np.float32(soft)), float(np.float32(hard))
    it = 1.0 / float(np.float32(temperature))
    loss, lerr = np.zeros(rows), np.zeros(rows)
    grad, tgrad = np.zeros(z.shape), np.zeros(z.shape)
    for r in np.flatnonzero(live):
        x = z[r:r + 1].astype(np.float64)
        w = float(weights[r]) if weights is not None else 1.0
        u = unit(x, it)[0, 0]
        keep = ids[r].astype(np.int64) < cols
        t = teacher[r][keep].astype(np.float64) * it
        fin = np.isfinite(t)
        span = float(t[fin].max() - t[fin].min()) if fin.any() else 0.0
        uq = HALF_STEP * (6 * min(span, 110.0) + len(t) + 60.0)           # the same bound for the list's own softmax
        if lse is not None:
            lq = t - float(lse[r])
            uq += HALF_STEP * 4
        else:
            lq = t - (t[fin].max() + np.log(np.exp(t[fin] - t[fin].max()).sum())) if fin.any() else np.full(t.shape, -np.inf)
        q = np.exp(lq)
        where = ids[r][keep].astype(np.int64)
        lp = log_softmax(x * it)[0]
        pos = q > 0
        l = float((q[pos] * (lq[pos] - lp[where[pos]])).sum())
        size = float((q[pos] * (np.abs(lq[pos]) + np.abs(lp[where[pos]]))).sum())
        mass = q.sum()
        qz = np.zeros(cols)
        np.add.at(qz, where, q)
        p = np.exp(lp)
        g = soft * it * (mass * p - qz)
        tg = abs(soft) * it * (2 * (u + uq) * mass * p + 2 * (uq + HALF_STEP * 4) * qz + (2 * u * mass * p) * (qz > 0))
        loss[r] = soft * l
        lerr[r] = abs(soft) * (uq * (size + mass) * 2 + u * mass)
        if hard and targets[r] < cols:
            lp1 = log_softmax(x)[0]
            u1 = unit(x)[0, 0]
            onehot = np.zeros(cols)
            onehot[targets[r]] = 1.0
            loss[r] -= hard * lp1[targets[r]]
            lerr[r] += abs(hard) * u1
            g = g + hard * (np.exp(lp1) - onehot)
            tg = tg + abs(hard) * 2 * u1 * (np.exp(lp1) + onehot)
        loss[r] *= w
        lerr[r] = abs(w) * lerr[r] + HALF_STEP * abs(loss[r])
        grad[r], tgrad[r] = g * w * scale, tg * abs(w) * scale
    return dict(loss=loss, grad=grad), dict(loss=lerr + 1e-38, grad=tgrad + 1e-38)
