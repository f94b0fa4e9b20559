"""Plain 64-bit forms of the operators on rows of logits, for the tests: numpy, row by row, nothing shared with the
engine. Every function returns the magnitudes that its error bounds are made of beside the values."""
import numpy as np

#: relative distance to the nearest value of a type, at most
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float64": 2.0 ** -53}
#: half the distance between a type's smallest values
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float64": 0.0}

# Relative error of a sum of a row's softmax terms in single precision. A term 2^d: ex2 is good to 2^-22; its argument
# d = x*kappa - shift carries two roundings of 2^-24 |d|, which a term weighs by p, and sum p |d| <= log2 V + 2 <= 19:
# 19 * 2 * 2^-24 * ln 2 < 2^-19. A thread adds at most 128 terms of a register-held row one after the other, a CTA's
# thread a 256th of a long one (70 000 / 256 = 274), then 8 levels of pairs: below 300 * 2^-24 < 2^-15.7 were every
# rounding to go the same way. Together below 2^-15.
# A single term is off by less: |d| < 126 where it is not zero, so 126 * 2 * 2^-24 * ln 2 + 2^-22 < 2^-16.
SUM32 = 2.0 ** -15
SUM64 = 1e-12

#: single-precision probabilities below 2^-126 are zero (ex2 flushes them), at the coefficients they are multiplied by
FLUSH32 = 2.0 ** -126


def row_softmax(x, tau):
    """(log-probabilities, probabilities) of one row; -inf / 0 where the row has no finite entry."""
    z = np.asarray(x, np.float64) / tau
    if np.isnan(z).any() or (z == np.inf).any():
        return np.full_like(z, np.nan), np.full_like(z, np.nan)
    m = z.max()
    if m == -np.inf:
        return np.full_like(z, -np.inf), np.zeros_like(z)
    lp = (z - m) - np.log(np.exp(z - m).sum())
    return lp, np.exp(lp)


def scores(x, targets, k, tau):
    """(log_probs [R,P], entropy [R], top_log_probs [R,k], top_indices [R,k]) in double."""
    R, V = x.shape
    P = 0 if targets is None else targets.shape[1]
    lps, ent, top, idx = np.zeros((R, P)), np.zeros(R), np.zeros((R, k)), np.zeros((R, k), np.int64)
    for r in range(R):
        lp, p = row_softmax(x[r], tau)
        for i in range(P):
            t = targets[r, i]
            lps[r, i] = 0.0 if t < 0 else np.nan if t >= V else lp[t]
        live = p > 0
        ent[r] = np.nan if np.isnan(lp).any() else -(p[live] * lp[live]).sum()
        # NaN first, then by value, the lower index first
        order = sorted(range(V), key=lambda j: (not np.isnan(x[r, j]), -x[r, j] if not np.isnan(x[r, j]) else 0.0, j))
        idx[r] = order[:k]
        top[r] = lp[idx[r]]
    return lps, ent, top, idx


def scores_grad(x, targets, idx, g_lp, g_ent, g_top, tau):
    """(gradient, magnitude, coefficient): the magnitude adds up the absolute values of the terms, the coefficient is
    what the probabilities are multiplied by."""
    R, V = x.shape
    grad, mag, coef = np.zeros((R, V)), np.zeros((R, V)), np.zeros((R, 1))
    for r in range(R):
        lp, p = row_softmax(x[r], tau)
        if (lp == -np.inf).all():
            continue
        picked = []
        if g_lp is not None:
            picked += [(t, g) for t, g in zip(targets[r], g_lp[r]) if 0 <= t < V]
        if g_top is not None:
            picked += list(zip(idx[r], g_top[r]))
        for t, g in picked:
            grad[r, t] += g
            mag[r, t] += abs(g)
        total = sum(g for _, g in picked)
        grad[r] -= p * total
        mag[r] += p * sum(abs(g) for _, g in picked)
        coef[r] += sum(abs(g) for _, g in picked)
        if g_ent is not None:
            lp0 = np.where(p > 0, lp, 0.0)
            h = -(p * lp0).sum()
            grad[r] -= g_ent[r] * p * (lp0 + h)
            mag[r] += abs(g_ent[r]) * p * (abs(lp0) + h)
            coef[r] += abs(g_ent[r]) * (100.0 + h)  # |ln p| of what is just flushed: below 100
    return grad / tau, mag / tau, coef / tau


def distill(x, teacher, index, weight, tail, tau):
    """(row losses, gradient rows of the sum, magnitudes of both) in double."""
    R, V = x.shape
    loss, grad = np.zeros(R), np.zeros((R, V))
    lmag, gmag = np.zeros(R), np.zeros((R, V))
    for r in range(R):
        w = 1.0 if weight is None else float(weight[r])
        if w == 0.0:
            continue
        entries = [(int(c), float(a)) for c, a in zip(index[r], teacher[r]) if c >= 0]
        lp, p = row_softmax(x[r], tau)
        if any(c >= V for c, _ in entries) or np.isnan(lp).any():
            loss[r], grad[r] = np.nan, np.nan
            continue
        if (lp == -np.inf).all():
            continue
        a = np.array([v for _, v in entries])
        if tail:
            q, lq = np.exp(a), a
        elif len(a) and a.max() > -np.inf:
            z = a / tau
            lq = z - (z.max() + np.log(np.exp(z - z.max()).sum()))
            q = np.exp(lq)
        else:
            q, lq = np.zeros(len(a)), np.full(len(a), -np.inf)
        D = M = 0.0
        Q = q.sum()
        for (c, _), qi, li in zip(entries, q, lq):
            if qi > 0:
                D += qi * (li - lp[c])
                M += qi * (abs(li) + abs(lp[c]) + 1.0)
        if tail:
            other = np.ones(V, bool)
            other[[c for c, _ in entries]] = False
            other &= x[r] > -np.inf
            if other.any():
                z = x[r] / tau
                part = np.exp(z[other] - z[other].max())
                lr = (z[other].max() - z.max()) + np.log(part.sum()) - np.log(np.exp(z - z.max()).sum())
                left = max(0.0, 1.0 - Q)
                Q += left
                if left > 0:
                    D += left * (np.log(left) - lr)
                    M += left * (abs(np.log(left)) + abs(lr) + 1.0)
                grad[r, other] -= left * part / part.sum()
                gmag[r, other] += left * part / part.sum()
        grad[r] += Q * p
        gmag[r] += Q * p
        for (c, _), qi in zip(entries, q):
            grad[r, c] -= qi
            gmag[r, c] += qi
        grad[r] *= w / tau
        gmag[r] *= abs(w) / tau
        loss[r], lmag[r] = w * D, abs(w) * M
    return loss, grad, lmag, gmag
