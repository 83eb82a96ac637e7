"""The operators on rows of category scores in 64 bits, row by row from their definitions, and what an implementation in 32 bits
may be off: shared by the CPU and the GPU tests."""
import numpy as np

EPS = 2.0 ** -24                                    # half a step of float32, relative
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}    # of the types, relative
TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}  # half of the smallest step, absolute
LOWEST = {"float32": -3.4028234663852886e38, "bfloat16": -3.3895313892515355e38, "float16": -65504.0}


def seen(x, dtype):
    """x with its masked scores, at or below half of the type's lowest value, at -inf"""
    return np.where(x <= LOWEST[dtype] / 2, -np.inf, x)


def _shifted(x):
    """Scores above the row's largest, and log Z above it: small numbers, whatever the level of the row"""
    m = x.max(1)
    bad = np.isnan(x).any(1) | (m == np.inf)
    safe = np.where(np.isfinite(m), m, 0.0)
    return safe, x - safe[:, None], np.log(np.exp(x - safe[:, None]).sum(1)), bad


def statistics(x):
    """log Z, entropy [rows] of x [rows, C] (float64 holding the scores' values)"""
    with np.errstate(all="ignore"):
        safe, d, ls, bad = _shifted(x)
        lp = d - ls[:, None]
        p = np.exp(lp)
        h = -np.where(p > 0, p * lp, 0.0).sum(1)
        z = safe + ls
        h[ls == -np.inf] = np.nan                    # no distribution
        z[bad] = np.nan
        h[bad] = np.nan
    return z, h


def logp_of(x, g):
    """log-probabilities of given categories g [rows, slots]"""
    C = x.shape[1]
    with np.errstate(all="ignore"):
        _, d, ls, bad = _shifted(x)
        lp = np.take_along_axis(d, np.clip(g, 0, C - 1), 1) - ls[:, None]
    lp = np.where(ls[:, None] == -np.inf, -np.inf, lp)
    lp = np.where(bad[:, None], np.nan, lp)
    return np.where(g < 0, 0.0, np.where(g >= C, np.nan, lp))


def likeliest(x, top):
    index = np.full((x.shape[0], top), -1, np.int64)
    logp = np.full((x.shape[0], top), -np.inf)
    with np.errstate(all="ignore"):
        _, d, ls, bad = _shifted(x)
    for r in range(x.shape[0]):
        if bad[r]:
            logp[r] = np.nan
            continue
        order = np.argsort(-x[r], kind="stable")[:top]
        order = order[x[r][order] > -np.inf]
        index[r, :len(order)] = order
        logp[r, :len(order)] = d[r][order] - ls[r]
    return index, logp


def gradient(x, z, h, slots, gh=None):
    """slots: pairs (categories [rows, k], derivatives [rows, k]); z, h as given (float64 of float32 values).  Returns the
    gradient, the size of its terms, which roundings are relative to, and what underflow may take away: a p below 2^-126, the
    smallest normal number of 32 bits, may count as 0, and with it its product with the rest of its term."""
    R, C = x.shape
    out = np.zeros((R, C))
    size = np.zeros((R, C))
    with np.errstate(all="ignore"):
        d = x - z[:, None]
        p = np.exp(d)
        total, weight = np.zeros(R), np.zeros(R)
        for g, w in slots:
            for j in range(g.shape[1]):
                for r in np.flatnonzero(g[:, j] >= 0):
                    total[r] += w[r, j] if g[r, j] < C else np.nan
                    weight[r] += abs(w[r, j])
                    if g[r, j] < C:
                        out[r, g[r, j]] += w[r, j]
                        size[r, g[r, j]] += abs(w[r, j])
        out -= p * total[:, None]
        # p is exp of a difference that is rounded at the size of its two terms
        slack = 1.0 + np.where(np.isfinite(d), np.abs(np.where(np.isfinite(x), x, 0.0)) + np.abs(z[:, None]), 0.0)
        size += p * weight[:, None] * slack
        under = np.broadcast_to(weight[:, None], out.shape).copy()
        if gh is not None:
            h = np.nan_to_num(h)
            out -= np.where(p > 0, gh[:, None] * p * (d + h[:, None]), 0.0)
            term = np.abs(gh[:, None]) * (np.minimum(np.abs(d), 200.0) + np.abs(h[:, None]) + 1.0)
            size += np.where(p > 0, p * term * slack, 0.0)
            under += term
    out[z == -np.inf] = 0.0
    size[z == -np.inf] = 0.0
    return out, size, 2.0 ** -126 * np.nan_to_num(under)


def rounded(x, dtype):
    """x [rows, C] as 8 bits hold it, block by block (dtype: name of the rows' type)"""
    out = np.empty_like(x)
    for r in range(x.shape[0]):
        for s in range(0, x.shape[1], 64):
            b = x[r, s:s + 64]
            if np.isnan(b).any() or (b == np.inf).any():
                out[r, s:s + 64] = np.nan
                continue
            off = b <= LOWEST[dtype] / 2
            k = b[~off]
            e = -126
            if len(k):
                f, q = np.frexp(np.float64(np.float32(k.max() - k.min())) if abs(k.max() - k.min()) < 3e38 else k.max() - k.min())
                if f > 0:
                    e = max(e, int(q) - (8 if f <= 253 / 256 else 7))
                a = np.abs(k).max()
                if a > 0:
                    e = max(e, int(np.frexp(a)[1]) - 14)
            step = 2.0 ** e
            out[r, s:s + 64] = np.where(off, -np.inf, np.minimum(np.rint(np.where(off, 0, b) / step) * step, -LOWEST["float32"]))
    return out


def sum_bound(C):
    """Relative error of the sum of C exponentials in 32 bits, each off by the rounding of its argument (at most 104 where it
    counts, times 2^-24, and as much again for the base's change), two units of the exponential, and one rounding per
    addition of a chain of C / 64 with 12 more to join lanes and parts"""
    return (2 * 104 + 4 + C / 64 + 12) * EPS


def log_bound(x, z, C):
    """Absolute error of a log-probability or of log Z: the sum's relative error, roundings of the logarithm and of terms"""
    m = np.nan_to_num(np.abs(np.where(np.isfinite(x), x, 0.0)).max(1), posinf=0.0)
    return sum_bound(C) + 4 * EPS * (m + np.nan_to_num(np.abs(z), posinf=0.0) + 20.0)


def entropy_bound(x, z, C):
    """log Z - t / Z: the error of the sums times the largest of their terms, log C"""
    return (sum_bound(C) + 8 * EPS) * (2.0 + 2.0 * np.log(C + 1.0))
