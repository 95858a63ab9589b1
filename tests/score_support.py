"""What the CPU and the GPU tests of the scoring ops share: inputs, the
oracle's answers and the tolerances."""
import ctypes

import numpy as np

from support import BF16, FP16, FP32, FTZ_LIMIT, U32, gamma, normal, oracle, ptr, rng, to_f64, to_storage, ulp

NO_TOKEN = 0xFFFFFFFF
DTS = [FP32, FP16, BF16]
DT_IDS = {FP32: "fp32", FP16: "fp16", BF16: "bf16"}


def dt_id(dt):
    return DT_IDS[dt]


def score_oracle():
    O = oracle()
    i, u64, f32, vp = ctypes.c_int, ctypes.c_uint64, ctypes.c_float, ctypes.c_void_p
    O.oracle_token_logprobs.argtypes = [i, i, i, u64, f32, i, i] + [vp] * 7
    O.oracle_token_logprobs_bwd.argtypes = [i, i, i, u64, f32, i] + [vp] * 7
    O.oracle_distillation_loss.argtypes = [i, i, i, u64, f32, i] + [vp] * 7
    return O


def logits(seed, shape, stride, dt, std=2.5, mean=0.0):
    """rows of a trained model's kind: a spread, an offset of each row's own,
    one column well above; the elements between the rows are NaN"""
    n_rows, n_cols = shape
    g = rng(seed)
    x = (mean + std * g.standard_normal(shape) + 2.0 * g.standard_normal((n_rows, 1))).astype(np.float32)
    x[np.arange(n_rows), g.integers(0, n_cols, n_rows)] += g.uniform(2.0, 16.0, n_rows).astype(np.float32)
    full = np.full((n_rows, stride), np.nan, np.float32)
    full[:, :n_cols] = x
    return to_storage(full, dt)


def want_logprobs(dt, x, n_cols, scale, tokens, top_k):
    n_rows, stride = x.shape
    M = tokens.shape[1]
    w = dict(logprobs=np.empty((n_rows, M)), entropy=np.empty(n_rows), lse=np.empty(n_rows),
             top_ids=np.zeros((n_rows, top_k), np.uint32), top_logprobs=np.empty((n_rows, top_k)))
    assert score_oracle().oracle_token_logprobs(dt, n_rows, n_cols, stride, scale, M, top_k, ptr(x), ptr(tokens),
                                                *[ptr(w[n]) for n in ("logprobs", "entropy", "lse", "top_ids", "top_logprobs")]) == 0
    return w


def want_grad(dt, x, n_cols, scale, tokens, lse, entropy, d_logprobs, d_entropy):
    n_rows, stride = x.shape
    dx = np.empty((n_rows, n_cols))
    assert score_oracle().oracle_token_logprobs_bwd(dt, n_rows, n_cols, stride, scale, tokens.shape[1], ptr(x), ptr(tokens), ptr(lse),
                                                    ptr(entropy), ptr(d_logprobs), ptr(d_entropy), ptr(dx)) == 0
    return dx


def want_distill(dt, x, n_cols, scale, ids, values, weights, grad=True):
    n_rows, stride = x.shape
    loss, mean, dx = np.empty(n_rows), np.zeros(1), np.empty((n_rows, n_cols)) if grad else None
    assert score_oracle().oracle_distillation_loss(dt, n_rows, n_cols, stride, scale, ids.shape[1], ptr(x), ptr(ids), ptr(values),
                                                   ptr(weights), ptr(loss), ptr(mean), ptr(dx)) == 0
    return loss, mean, dx


# ---------------- tolerances ----------------
#
# u = 2^-24. A term of Z is exp2(d * (s log2 e)) with d = x - M: the difference,
# the constant, the product and exp2 (one ulp) are off by at most
# (4 |s d| + 2) u of the term, and E's terms by 2 u more. The sums run over at
# most min(n / 64, 160) + 40 additions for any term. Weighted with p, |s d| is
# |E| / Z = log Z - entropy <= log n.

def depth(n_cols):
    return min(n_cols // 64, 160) + 40


def z_slack(n_cols):
    """relative error of Z, and so the absolute one of log Z (whose own
    rounding, of a value up to log n, is in too)"""
    return gamma(depth(n_cols)) + (6.0 * np.log(max(n_cols, 2)) + 4.0) * U32


def logprob_tol(n_cols, lp):
    """s (x - M) - log Z: the two roundings of its first part, |lp| + log n at
    most, and of the difference"""
    return z_slack(n_cols) + 4.0 * (np.abs(lp) + np.log(max(n_cols, 2))) * U32


def entropy_tol(n_cols):
    """log Z - E / Z: log Z's error, and E / Z (at most log n) with the
    relative errors of E and of Z"""
    return z_slack(n_cols) * (1.0 + 2.0 * np.log(max(n_cols, 2))) + 4.0 * np.log(max(n_cols, 2)) * U32


def close(o, v, tol, what):
    """fp32 results against their values in 64 bits: infinities and NaN in the
    same places, the rest within tol (absolute) and the rounding of the result"""
    o, v = np.asarray(o, np.float64), np.asarray(v, np.float64)
    tol = np.broadcast_to(np.asarray(tol, np.float64), v.shape)
    assert np.array_equal(np.isnan(o), np.isnan(v)), what + ": NaN in other places"
    inf = np.isinf(v)
    assert np.array_equal(o[inf], v[inf]) and not np.isinf(o[~inf]).any(), what + ": infinities in other places"
    fin = np.isfinite(v)
    off = np.abs(o[fin] - v[fin]) - (tol[fin] + np.abs(v[fin]) * U32)
    assert not (off > 0).any(), "%s: %d of %d off, worst by %g" % (what, (off > 0).sum(), off.size, off.max())


def rounded_once(o, dt, v, slack, what):
    """outputs of type dt: the rounding (half a step) of a value within `slack`
    of v; fp32's subnormal range may flush to zero. fp16 ends at 65504, so what
    lies half a step (16) beyond rounds to infinity, and only that."""
    of, v = to_f64(o, dt), np.asarray(v, np.float64)
    if dt == FP16:
        beyond = np.isinf(of)
        assert (np.sign(of) * v + slack)[beyond].min(initial=np.inf) >= 65520.0 and (np.abs(v) - slack)[~beyond].max(initial=0.0) < 65520.0 or np.isnan(v).any(), what
        of = np.where(beyond & np.isfinite(v), v, of)
    nan = np.isnan(v)
    assert np.array_equal(np.isnan(of), nan), what + ": NaN in other places"
    off = np.abs(of - v) - (0.5 * ulp(np.abs(v) + slack, dt) + slack + 2.0 * FTZ_LIMIT)
    bad = (off > 0) & ~nan
    assert not bad.any(), "%s: %d of %d off, first at %s: %r for %r" % (what, bad.sum(), bad.size, np.argwhere(bad)[0], of[bad][0], v[bad][0])


def grad_slack(dt, x, n_cols, scale, tokens, lse, entropy, d_logprobs, d_entropy):
    """fp32 evaluation of s (g - p (G + h (log p + H))): p is off by
    (4 |log p| + 6) u, G by gamma(M) of the sum of |g|, each product and sum by u"""
    xf = to_f64(x, dt)[:, :n_cols]
    s = float(np.float32(scale))
    with np.errstate(all="ignore"):
        lp = s * xf - lse.astype(np.float64)[:, None]
        p = np.exp(lp)
        there = tokens < n_cols
        gabs = np.abs(np.where(there, d_logprobs, 0.0)).sum(1, keepdims=True)
        f = gabs.copy() * np.ones_like(p)
        if d_entropy is not None:
            f = f + np.abs(d_entropy.astype(np.float64))[:, None] * (np.abs(lp) + np.abs(entropy.astype(np.float64))[:, None])
        sl = np.where(p > 0, s * p * f * (4.0 * np.abs(lp) + 12.0 + 2.0 * tokens.shape[1]) * U32, 0.0)
    rows, m = np.nonzero(there)
    extra = np.zeros_like(sl)
    np.add.at(extra, (rows, tokens[rows, m]), s * np.abs(d_logprobs[rows, m].astype(np.float64)) * (tokens.shape[1] + 4) * U32)
    return np.nan_to_num(sl + extra, nan=0.0, posinf=0.0)


def distill_slack(dt, x, n_cols, scale, ids, weights):
    """fp32 evaluation of w T (p - q): p is off by Z's error and
    (4 |log p| + 8) u, the sum of a column's q's by the teacher's sum (K terms)
    and (4 (s |v - max|) + 8) u, of which q at most 1"""
    xf = to_f64(x, dt)[:, :n_cols]
    s = float(np.float32(scale))
    with np.errstate(all="ignore"):
        z = s * (xf - xf.max(1, keepdims=True))
        lp = z - np.log(np.exp(z).sum(1, keepdims=True))
        p = np.exp(lp)
        sl = np.where(p > 0, p * (z_slack(n_cols) + (4.0 * np.abs(lp) + 12.0) * U32), 0.0)
    rows, k = np.nonzero(ids < n_cols)
    sl[rows, ids[rows, k]] += (2.0 * ids.shape[1] + 24.0) * U32
    return np.nan_to_num(sl, nan=0.0) * np.abs(np.float64(1.0) if weights is None else weights.astype(np.float64)[:, None]) / s


def distill_loss_tol(n_cols, scale, k):
    """T^2 sum q (log q - log p): q off by (2 K + 24) u, each difference of
    logarithms, at most a few tens, by logprob_tol and the teacher's like"""
    s = float(np.float32(scale))
    return (logprob_tol(n_cols, 64.0) + (2.0 * k + 24.0) * 64.0 * U32) / s ** 2


def tokens_for(seed, n_rows, n_cols, m, missing=True):
    t = rng(seed).integers(0, n_cols, (n_rows, m)).astype(np.uint32)
    if missing and m > 1:
        t[:, 1] = t[:, 0]          # the same token twice
    if missing and n_rows > 2 and m:
        t[2, 0] = NO_TOKEN         # no column
        t[1, m - 1] = n_cols       # the first that is none
    return t


def teacher_for(seed, n_rows, n_cols, k):
    g = rng(seed)
    ids = np.stack([g.permutation(n_cols)[:k] if k <= n_cols else g.integers(0, n_cols, k) for _ in range(n_rows)]).astype(np.uint32)
    v = (np.linspace(6.0, 0.0, k) + 1.5 * g.standard_normal((n_rows, k))).astype(np.float32)
    if k > 2:
        ids[:, 2] = ids[:, 0]      # the same column twice
        ids[0, k // 2:] = NO_TOKEN     # a short list
        v[-1, 1] = -np.inf
    return ids.reshape(n_rows, k), v


def normal_f32(seed, shape):
    return normal(seed, shape).astype(np.float32)
