"""The scoring ops on an AMD GPU through the C ABI, against their oracle in 64
bits: every storage type, row lengths from one column to hundreds of
thousands, odd lengths and strides, rows that masks leave empty, ties, the
calls that belong together, and calls that run beside each other."""
import ctypes
import threading

import numpy as np
import pytest

from score_support import (DTS, NO_TOKEN, close, distill_loss_tol, distill_slack, dt_id, entropy_tol, grad_slack, logits, logprob_tol, normal_f32,
                           rounded_once, teacher_for, tokens_for, want_distill, want_grad, want_logprobs, z_slack)
from support import BF16, ELEM_BYTES, FP16, FP32, NP_STORAGE, U32, rng, to_f64, to_storage
from test_hip_ops import Dev

from dataflow_lib_amd import api

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hdl():
    h = api.Handle(0, num_streams=2, scores=True)
    yield h
    h.destroy()


def space(d, nbytes):
    """a workspace of any content"""
    return (nbytes, d.put(np.full(nbytes, 0xAB, np.uint8))) if nbytes else (0, None)


def run_logprobs(h, dt, x, n_cols, scale, tokens, top_k, stream=0, offset=0, ws=True):
    n_rows, stride = x.shape
    M = tokens.shape[1]
    with Dev(h) as d:
        px, pt = d.put(x, offset * ELEM_BYTES[dt]), d.put(tokens)
        plp, pe, pl = d.put(np.full((n_rows, M), 7.0, np.float32)), d.empty(4 * n_rows), d.empty(4 * n_rows)
        pi, pv = d.put(np.full((n_rows, top_k), 7, np.uint32)), d.put(np.full((n_rows, top_k), 7.0, np.float32))
        sp = space(d, api.token_logprobs_workspace(dt, n_rows, n_cols, top_k))
        assert api.submit_token_logprobs(h, stream, dt, n_rows, n_cols, stride, scale, M, top_k, px, pt, plp, pe, pl, pi, pv, *sp) == 0
        return dict(logprobs=d.get(plp, (n_rows, M), np.float32), entropy=d.get(pe, (n_rows,), np.float32), lse=d.get(pl, (n_rows,), np.float32),
                    top_ids=d.get(pi, (n_rows, top_k), np.uint32), top_logprobs=d.get(pv, (n_rows, top_k), np.float32))


def check_logprobs(dt, x, n_cols, scale, tokens, top_k, got, what=""):
    w = want_logprobs(dt, x, n_cols, scale, tokens, top_k)
    assert np.array_equal(got["top_ids"], w["top_ids"]), what + ": top ids"
    with np.errstate(invalid="ignore"):
        close(got["logprobs"], w["logprobs"], logprob_tol(n_cols, w["logprobs"]), what + " logprobs")
        close(got["top_logprobs"], w["top_logprobs"], logprob_tol(n_cols, w["top_logprobs"]), what + " top logprobs")
        close(got["lse"], w["lse"], z_slack(n_cols) + 2.0 * np.abs(w["lse"]) * U32, what + " lse")
    close(got["entropy"], w["entropy"], entropy_tol(n_cols), what + " entropy")
    return w


# rows, columns, columns between rows, elements off the alignment, tokens, top k
SHAPES = [(1, 1, 0, 0, 1, 1), (3, 2, 1, 1, 2, 2), (5, 7, 0, 0, 1, 7), (7, 64, 0, 0, 3, 8), (9, 65, 3, 0, 2, 65), (33, 1000, 0, 0, 1, 20), (300, 255, 1, 3, 1, 5),
          (17, 2049, 0, 5, 4, 64), (70, 8192, 0, 0, 1, 1), (5, 16385, 15, 0, 1, 128), (64, 32000, 64, 0, 4, 10), (4, 50257, 0, 0, 1, 256), (600, 4099, 0, 0, 1, 40),
          (2, 128256, 0, 0, 1, 20), (1, 151937, 0, 1, 1, 100), (3, 300001, 7, 0, 5, 256), (130, 65537, 0, 0, 1, 0), (257, 40000, 0, 0, 0, 3), (12, 131072, 0, 8, 1, 33),
          (2500, 300, 20, 0, 1, 7), (1, 1 << 21, 0, 0, 2, 50), (1, 1 << 21, 1, 0, 1, 256), (2, 128257, 0, 0, 3, 0), (60, 1000, 0, 0, 1, 256),
          (90, 513, 0, 1, 1, 30), (1030, 6001, 1, 0, 1, 20), (600, 4096, 0, 0, 1, 100), (700, 20001, 0, 3, 1, 256), (2100, 1500, 0, 0, 2, 250)]


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d+%d_off%d_m%d_k%d" % s)
def test_token_logprobs(hdl, dt, shape):
    n_rows, n_cols, pad, off, m, k = shape
    scale = (1.0, 0.7, 2.0)[n_cols % 3]
    x, tok = logits(n_cols, (n_rows, n_cols), n_cols + pad, dt), tokens_for(n_rows, n_rows, n_cols, m)
    got = run_logprobs(hdl, dt, x, n_cols, scale, tok, k, offset=off)
    check_logprobs(dt, x, n_cols, scale, tok, k, got, "%dx%d" % (n_rows, n_cols))


def odd_rows(n_cols, dt):
    """rows by kind: all equal, -inf alone, one column above -inf, the type's
    lowest value alone, lowest and a few, NaN in one place, NaN alone, +inf,
    +-0, sorted rising, sorted falling, few values (ties), far from zero both
    ways, a huge range"""
    g = rng(n_cols)
    low = float(np.finfo(np.float16).min) if dt == FP16 else float(to_f64(np.array([0xFF7F], np.uint16), BF16)[0]) if dt == BF16 else float(np.finfo(np.float32).min)
    big = 6.0e4 if dt == FP16 else 1.0e38
    base = g.standard_normal(n_cols) * 2.5
    some = g.permutation(n_cols)[:max(1, n_cols // 100)]
    rows = [np.full(n_cols, 3.25), np.full(n_cols, -np.inf), np.full(n_cols, -np.inf), np.full(n_cols, low), np.full(n_cols, low), base.copy(),
            np.full(n_cols, np.nan), base.copy(), np.where(g.random(n_cols) < 0.5, 0.0, -0.0), np.sort(base), -np.sort(-base), g.integers(0, 3, n_cols) * 1.0,
            base + 300.0, base - 300.0, np.linspace(-big, big, n_cols), np.full(n_cols, -np.inf), base * 1e-3]
    rows[2][n_cols // 2] = -5.0
    rows[4][some] = base[some]
    rows[5][n_cols - 1] = np.nan
    rows[7][n_cols // 3] = np.inf
    rows[15][some] = base[some]
    return to_storage(np.array(rows, np.float32), dt)


ODD_LENGTHS = [3, 66, 1000, 4099, 20000, 50257, 131080, 300001]


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("n_cols", ODD_LENGTHS)
def test_token_logprobs_of_odd_rows(hdl, dt, n_cols):
    x = odd_rows(n_cols, dt)
    tok = tokens_for(5, len(x), n_cols, 2)
    k = min(n_cols, 60)
    got = run_logprobs(hdl, dt, x, n_cols, 1.0, tok, k)
    w = want_logprobs(dt, x, n_cols, 1.0, tok, k)
    assert np.array_equal(got["top_ids"], w["top_ids"])
    with np.errstate(invalid="ignore"):
        for name in ("logprobs", "top_logprobs"):
            close(got[name], w[name], logprob_tol(n_cols, w[name]), name)
        close(got["lse"], w["lse"], z_slack(n_cols) + 2.0 * np.abs(w["lse"]) * U32, "lse")
    close(got["entropy"], w["entropy"], entropy_tol(n_cols), "entropy")


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("n_cols,k", [(50257, 20), (128256, 200), (5000, 256), (700000, 64)])
def test_top_ids_where_the_largest_lie_together(hdl, dt, n_cols, k):
    """the largest logits in one block, all above the rest; the same over many
    rows, with blocks at the row's ends, and ties across the k-th place"""
    g = rng(k)
    rows = []
    for first in (0, n_cols // 2, n_cols - 3 * k):
        r = g.standard_normal(n_cols)
        r[first:first + 3 * k] = 20.0 + g.permutation(3 * k) * 0.125
        rows.append(r)
        t = g.standard_normal(n_cols)
        t[first:first + 3 * k] = 8.0
        rows.append(t)
    x = to_storage(np.array(rows, np.float32), dt)
    tok = tokens_for(6, len(x), n_cols, 1)
    got = run_logprobs(hdl, dt, x, n_cols, 1.0, tok, k)
    check_logprobs(dt, x, n_cols, 1.0, tok, k, got)


def test_operands_left_out(hdl):
    n_rows, n_cols = 5, 3000
    x = logits(20, (n_rows, n_cols), n_cols, BF16)
    w = want_logprobs(BF16, x, n_cols, 1.0, tokens_for(1, n_rows, n_cols, 1), 3)
    with Dev(hdl) as d:
        px, pl, pe = d.put(x), d.empty(4 * n_rows), d.empty(4 * n_rows)
        pi, pv = d.empty(12 * n_rows), d.empty(12 * n_rows)
        sp = space(d, api.token_logprobs_workspace(BF16, n_rows, n_cols, 3))
        call = lambda *a: api.submit_token_logprobs(hdl, 0, BF16, n_rows, n_cols, n_cols, 1.0, *a, *sp)  # noqa: E731
        assert call(0, 0, px, None, None, None, pl, None, None) == 0
        assert call(0, 0, px, None, None, pe, None, None, None) == 0
        assert call(0, 3, px, None, None, None, None, pi, pv) == 0
        assert call(0, 0, px, None, None, None, None, None, None) == 0
        close(d.get(pl, (n_rows,), np.float32), w["lse"], z_slack(n_cols) + 2.0 * np.abs(w["lse"]) * U32, "lse")
        close(d.get(pe, (n_rows,), np.float32), w["entropy"], entropy_tol(n_cols), "entropy")
        assert np.array_equal(d.get(pi, (n_rows, 3), np.uint32), w["top_ids"])


# ---------------- gradients ----------------

def forward_for(dt, x, n_cols, scale, tokens):
    w = want_logprobs(dt, x, n_cols, scale, tokens, 0)
    return w["lse"].astype(np.float32), w["entropy"].astype(np.float32)


def run_grad(h, dt, x, n_cols, scale, tok, lse, ent, g, he, grad_stride=None, offset=0, g_offset=0, in_place=False):
    """the whole gradient buffer, its gaps too"""
    n_rows, stride = x.shape
    grad_stride = stride if in_place else (grad_stride or n_cols)
    with Dev(h) as d:
        e = ELEM_BYTES[dt]
        px = d.put(x, offset * e)
        pd = px if in_place else d.put(to_storage(np.full((n_rows, grad_stride), 3.0, np.float32), dt), g_offset * e)
        args = [d.put(a) if a is not None else None for a in (tok, lse, ent, g, he)]
        assert api.submit_token_logprobs_bwd(h, 0, dt, n_rows, n_cols, stride, grad_stride, scale, tok.shape[1], px, *args, pd) == 0
        out = d.get(pd, (n_rows, grad_stride), NP_STORAGE[dt])
        if not in_place:
            assert np.array_equal(d.get(px, x.shape, NP_STORAGE[dt]).view(np.uint8), x.view(np.uint8)), "the logits were written"
        return out


# rows, columns, between rows of logits and of gradients, elements off the
# alignment of each, tokens
GRAD_SHAPES = [(1, 1, 0, 0, 0, 0, 1), (3, 2, 1, 0, 1, 0, 2), (5, 7, 0, 0, 0, 0, 1), (9, 65, 3, 1, 0, 0, 4), (33, 1000, 0, 0, 0, 0, 1), (300, 255, 0, 1, 3, 2, 2),
               (17, 2049, 0, 0, 5, 0, 32), (70, 8192, 0, 8, 0, 0, 1), (64, 32000, 64, 0, 0, 0, 3), (4, 50257, 0, 0, 0, 0, 1), (600, 4099, 0, 0, 0, 1, 2),
               (2, 128256, 0, 0, 0, 0, 1024), (1, 151937, 0, 0, 1, 0, 1), (3, 300001, 7, 0, 0, 0, 5), (2500, 300, 20, 4, 0, 0, 1), (130, 65537, 0, 0, 0, 0, 0)]


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("shape", GRAD_SHAPES, ids=lambda s: "%dx%d+%d+%d_off%d,%d_m%d" % s)
def test_token_logprobs_bwd(hdl, dt, shape):
    n_rows, n_cols, pad, gpad, off, goff, m = shape
    scale = (1.0, 0.7, 2.0)[n_cols % 3]
    x, tok = logits(n_cols, (n_rows, n_cols), n_cols + pad, dt), tokens_for(n_rows, n_rows, n_cols, m)
    lse, ent = forward_for(dt, x, n_cols, scale, tok)
    g, he = normal_f32(1, (n_rows, m)), normal_f32(2, (n_rows,))
    for h in (he, None) if m else (he,):
        e = ent if h is not None else None
        out = run_grad(hdl, dt, x, n_cols, scale, tok, lse, e, g, h, n_cols + gpad, off, goff)
        v = want_grad(dt, x, n_cols, scale, tok, lse, e, g, h)
        rounded_once(out[:, :n_cols], dt, v, grad_slack(dt, x, n_cols, scale, tok, lse, e, g, h), "dlogits")
        assert np.all(to_f64(out[:, n_cols:], dt) == 3.0), "columns behind the row were written"


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("shape", [(6, 257, 3, 1, 6), (3, 50257, 0, 0, 40), (400, 3001, 0, 0, 2), (2, 200000, 8, 3, 1000)], ids=lambda s: "%dx%d+%d_off%d_m%d" % s)
def test_token_logprobs_bwd_in_place(hdl, dt, shape):
    """the same bits as out of place, and the columns between rows untouched"""
    n_rows, n_cols, pad, off, m = shape
    x, tok = logits(n_cols, (n_rows, n_cols), n_cols + pad, dt), tokens_for(n_rows, n_rows, n_cols, m)
    lse, ent = forward_for(dt, x, n_cols, 1.0, tok)
    g, he = normal_f32(1, (n_rows, m)), normal_f32(2, (n_rows,))
    apart = run_grad(hdl, dt, x, n_cols, 1.0, tok, lse, ent, g, he, n_cols + pad, off, off)
    inside = run_grad(hdl, dt, x, n_cols, 1.0, tok, lse, ent, g, he, offset=off, in_place=True)
    assert np.array_equal(inside[:, :n_cols].view(np.uint8), apart[:, :n_cols].view(np.uint8))
    assert np.array_equal(inside[:, n_cols:].view(np.uint8), x[:, n_cols:].view(np.uint8))


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("n_cols", ODD_LENGTHS)
def test_token_logprobs_bwd_of_odd_rows(hdl, dt, n_cols):
    x = odd_rows(n_cols, dt)
    tok = tokens_for(5, len(x), n_cols, 3)
    lse, ent = forward_for(dt, x, n_cols, 1.0, tok)
    g, he = normal_f32(1, tok.shape), normal_f32(2, (len(x),))
    g[9], he[9] = 0.0, 0.0           # nothing comes down: a row of zeros
    g[6], he[6] = 0.0, 0.0           # also where the logits are NaN
    with np.errstate(over="ignore"):
        v = want_grad(dt, x, n_cols, 1.0, tok, lse, ent, g, he)
        slack = grad_slack(dt, x, n_cols, 1.0, tok, lse, ent, g, he)
    out = run_grad(hdl, dt, x, n_cols, 1.0, tok, lse, ent, g, he)
    rounded_once(out, dt, v, slack, "dlogits of odd rows")
    assert not to_f64(out, dt)[[1, 6, 9]].any()


@pytest.mark.parametrize("dt", [FP32, BF16], ids=dt_id)
@pytest.mark.parametrize("scale, down", [(1.0, 1e9), (1e6, 1e4)])
def test_large_gradients_of_masked_rows(hdl, dt, scale, down):
    """columns of -inf get gradient 0 however large the entropy's gradient is"""
    n_rows, n_cols = 3, 5003
    x = logits(150, (n_rows, n_cols), n_cols, dt)
    xf = to_f64(x, dt)
    xf[:, ::3] = -np.inf
    xf[:, 101] = xf[:, 100] = xf[np.isfinite(xf)].max() + 1.0   # two share all that the larger scale leaves
    x = to_storage(xf.astype(np.float32), dt)
    tok = tokens_for(151, n_rows, n_cols, 1)
    lse, ent = forward_for(dt, x, n_cols, scale, tok)
    g, he = normal_f32(152, (n_rows, 1)), np.float32(down) * np.array([1.0, -1.0, 0.5], np.float32)
    out = run_grad(hdl, dt, x, n_cols, scale, tok, lse, ent, g, he)
    o = to_f64(out, dt)
    here = np.ones(n_cols, bool)
    here[tok[tok < n_cols]] = False
    assert np.isfinite(o).all() and not o[:, ~np.isfinite(xf[0]) & here].any()
    if scale == 1.0:
        v = want_grad(dt, x, n_cols, scale, tok, lse, ent, g, he)
        rounded_once(out, dt, v, grad_slack(dt, x, n_cols, scale, tok, lse, ent, g, he), "dlogits")


def test_gradient_against_differences(hdl):
    """the kernels alone: the loss through token_logprobs at shifted logits
    against token_logprobs_bwd, fp32"""
    n_cols, m, step = 50, 3, 2.0 ** -6
    x = logits(30, (1, n_cols), n_cols, FP32, std=1.0)
    tok, g, he = tokens_for(31, 1, n_cols, m, missing=False), normal_f32(32, (1, m)), normal_f32(33, (1,))
    shifted = np.concatenate([x + step * np.eye(n_cols, dtype=np.float32), x - step * np.eye(n_cols, dtype=np.float32), x])
    got = run_logprobs(hdl, FP32, shifted, n_cols, 0.5, np.repeat(tok, len(shifted), 0), 0)
    loss = (got["logprobs"].astype(np.float64) * g).sum(1) + got["entropy"].astype(np.float64) * he[0]
    numeric = (loss[:n_cols] - loss[n_cols:2 * n_cols]) / (2 * step)
    dx = run_grad(hdl, FP32, x, n_cols, 0.5, tok, got["lse"][-1:], got["entropy"][-1:], g, he)
    # third derivatives are below 1 here: step^2 / 6, and 1e-6 of fp32 noise over 2 steps
    assert np.abs(dx[0] - numeric).max() < step ** 2 / 6 + 4e-6 * (np.abs(g).sum() + 1) / step


# ---------------- distillation ----------------

def run_distill(h, dt, x, n_cols, scale, ids, v, wt, grad=True, mean=True, grad_stride=None, offset=0, g_offset=0, in_place=False, stream=0):
    n_rows, stride = x.shape
    K = ids.shape[1]
    grad_stride = stride if in_place else (grad_stride or n_cols)
    with Dev(h) as d:
        e = ELEM_BYTES[dt]
        px = d.put(x, offset * e)
        pd = None if not grad else px if in_place else d.put(to_storage(np.full((n_rows, grad_stride), 3.0, np.float32), dt), g_offset * e)
        pi, pv, pw = d.put(ids), d.put(v), d.put(wt) if wt is not None else None
        pl, pm = d.put(np.full(n_rows, 7.0, np.float32)), d.put(np.full(1, 7.0, np.float32)) if mean else None
        sp = space(d, api.distillation_loss_workspace(dt, n_rows, n_cols, K))
        assert api.submit_distillation_loss(h, stream, dt, n_rows, n_cols, stride, grad_stride, scale, K, px, pi, pv, pw, pl, pm, pd, *sp) == 0
        return d.get(pl, (n_rows,), np.float32), d.get(pm, (1,), np.float32) if mean else None, d.get(pd, (n_rows, grad_stride), NP_STORAGE[dt]) if grad else None


def check_distill(dt, x, n_cols, scale, ids, v, wt, got):
    loss, mean, out = got
    l, m, dx = want_distill(dt, x, n_cols, scale, ids, v, wt, grad=out is not None)
    tol = distill_loss_tol(n_cols, scale, ids.shape[1])
    close(loss, l, tol + np.abs(l) * 8 * U32, "loss")
    if mean is not None:
        w = np.ones(len(l)) if wt is None else np.abs(wt.astype(np.float64))
        close(mean, m, np.nan_to_num((w * (tol + np.nan_to_num(np.abs(l), posinf=0.0) * 8 * U32)).mean()), "mean loss")
    if out is not None:
        rounded_once(out[:, :n_cols], dt, dx, distill_slack(dt, x, n_cols, scale, ids, wt), "dlogits")
        assert np.all(to_f64(out[:, n_cols:], dt) == 3.0), "columns behind the row were written"


# rows, columns, between rows of logits and of gradients, elements off the
# alignment of each, teacher entries
KD_SHAPES = [(1, 1, 0, 0, 0, 0, 1), (3, 2, 1, 0, 1, 0, 2), (5, 7, 0, 0, 0, 0, 4), (9, 65, 3, 1, 0, 0, 65), (33, 1000, 0, 0, 0, 0, 8), (300, 255, 0, 1, 3, 2, 5),
             (17, 2049, 0, 0, 5, 0, 32), (70, 8192, 0, 8, 0, 0, 1), (64, 32000, 64, 0, 0, 0, 10), (4, 50257, 0, 0, 0, 0, 1024), (600, 4099, 0, 0, 0, 1, 64),
             (2, 128256, 0, 0, 0, 0, 64), (1, 151937, 0, 0, 1, 0, 100), (3, 300001, 7, 0, 0, 0, 50), (2500, 300, 20, 4, 0, 0, 16), (130, 65536, 0, 0, 0, 0, 20),
             (300, 131072, 0, 0, 0, 0, 16), (280, 65544, 0, 0, 8, 8, 64), (270, 32768, 0, 0, 0, 0, 128), (260, 131073, 0, 0, 0, 0, 3), (20, 70, 0, 0, 0, 0, 100),
             (70, 70001, 0, 0, 1, 0, 40)]


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("shape", KD_SHAPES, ids=lambda s: "%dx%d+%d+%d_off%d,%d_k%d" % s)
def test_distillation_loss(hdl, dt, shape):
    n_rows, n_cols, pad, gpad, off, goff, k = shape
    scale = (1.0, 0.5, 0.25)[n_cols % 3]
    x = logits(n_cols, (n_rows, n_cols), n_cols + pad, dt)
    ids, v = teacher_for(n_rows, n_rows, n_cols, k)
    wt = np.where(rng(3).random(n_rows) < 0.2, 0.0, rng(4).uniform(0.1, 2.0, n_rows)).astype(np.float32)
    check_distill(dt, x, n_cols, scale, ids, v, wt, run_distill(hdl, dt, x, n_cols, scale, ids, v, wt, grad_stride=n_cols + gpad, offset=off, g_offset=goff))
    got = run_distill(hdl, dt, x, n_cols, scale, ids, v, None, grad=False, offset=off)
    check_distill(dt, x, n_cols, scale, ids, v, None, got)


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("shape", [(6, 257, 3, 1, 6), (3, 50257, 0, 0, 40), (400, 3001, 0, 0, 2), (2, 200000, 8, 3, 1000), (300, 128256, 0, 0, 64)],
                         ids=lambda s: "%dx%d+%d_off%d_k%d" % s)
def test_distillation_in_place(hdl, dt, shape):
    """the same bits as out of place, and the columns between rows untouched"""
    n_rows, n_cols, pad, off, k = shape
    x = logits(n_cols, (n_rows, n_cols), n_cols + pad, dt)
    ids, v = teacher_for(n_rows, n_rows, n_cols, k)
    apart = run_distill(hdl, dt, x, n_cols, 0.5, ids, v, None, grad_stride=n_cols + pad, offset=off, g_offset=off)
    inside = run_distill(hdl, dt, x, n_cols, 0.5, ids, v, None, offset=off, in_place=True, mean=False)
    assert np.array_equal(inside[0], apart[0]) and inside[1] is None
    assert np.array_equal(inside[2][:, :n_cols].view(np.uint8), apart[2][:, :n_cols].view(np.uint8))
    assert np.array_equal(inside[2][:, n_cols:].view(np.uint8), x[:, n_cols:].view(np.uint8))


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("n_cols", ODD_LENGTHS + [128256])
def test_distillation_of_odd_rows(hdl, dt, n_cols):
    x = odd_rows(n_cols, dt)
    ids, v = teacher_for(7, len(x), n_cols, min(n_cols, 6))
    ids[8] = NO_TOKEN                # no teacher entry at all
    v[11] = -np.inf
    wt = np.ones(len(x), np.float32)
    wt[[6, 9]] = 0.0                 # not counted: zeros, also where the logits are NaN
    # probabilities of columns that a mask excludes make the loss infinite
    ids[[2, 4, 15, 14]] = NO_TOKEN
    got = run_distill(hdl, dt, x, n_cols, 1.0, ids, v, wt, mean=False)
    l, _, dx = want_distill(dt, x, n_cols, 1.0, ids, v, wt)
    close(got[0], l, distill_loss_tol(n_cols, 1.0, ids.shape[1]) + np.nan_to_num(np.abs(l), posinf=0.0) * 8 * U32, "loss")
    with np.errstate(invalid="ignore"):
        rounded_once(got[2], dt, dx, distill_slack(dt, x, n_cols, 1.0, ids, wt), "dlogits of odd rows")
    assert not to_f64(got[2], dt)[[1, 2, 4, 6, 8, 9, 11]].any() and not got[0][[2, 4, 6, 8, 9, 11]].any() and got[0][1] == np.inf


def test_teacher_values_that_are_no_numbers(hdl):
    """NaN and +inf among a teacher's values: NaN in that row, no other"""
    n_cols = 3000
    x = logits(40, (4, n_cols), n_cols, BF16)
    ids, v = teacher_for(41, 4, n_cols, 5)
    v[1, 0], v[2, 3] = np.nan, np.inf
    ids[1:3] = rng(42).permutation(n_cols)[:5]
    loss, _, dx = run_distill(hdl, BF16, x, n_cols, 1.0, ids, v, None, mean=False)
    assert np.array_equal(np.isnan(loss), [False, True, True, False])
    assert np.isnan(to_f64(dx, BF16)[1, ids[1]]).all() and np.isnan(to_f64(dx, BF16)[2, ids[2]]).all() and np.isfinite(to_f64(dx, BF16)[[0, 3]]).all()


# ---------------- the ops together, and beside each other ----------------

@pytest.mark.parametrize("dt", DTS, ids=dt_id)
def test_a_teacher_scores_and_a_student_learns(hdl, dt):
    """as they are used: the teacher's alternatives are written by one call and
    read by the next on the same stream, with nothing in between; the student's
    log-probabilities and their gradient come from its own forward pass"""
    n_rows, n_cols, k, s = 60, 32001, 40, 0.5
    t, x = logits(50, (n_rows, n_cols), n_cols, dt), logits(51, (n_rows, n_cols), n_cols, dt)
    tok, wt, g, he = tokens_for(52, n_rows, n_cols, 1), np.ones(n_rows, np.float32), normal_f32(53, (n_rows, 1)), normal_f32(54, (n_rows,))
    with Dev(hdl) as d:
        pt, px, ptok, pw, pg, ph = d.put(t), d.put(x), d.put(tok), d.put(wt), d.put(g), d.put(he)
        pi, pv, plp, pl, pe, ploss, pmean = (d.empty(n) for n in (4 * n_rows * k, 4 * n_rows * k, 4 * n_rows, 4 * n_rows, 4 * n_rows, 4 * n_rows, 4))
        pd, pk = d.empty(x.nbytes), d.empty(x.nbytes)
        s1, s2, s3 = (space(d, f(dt, n_rows, n_cols, q)) for f, q in ((api.token_logprobs_workspace, k), (api.token_logprobs_workspace, 0),
                                                                      (api.distillation_loss_workspace, k)))
        assert api.submit_token_logprobs(hdl, 0, dt, n_rows, n_cols, n_cols, 1.0, 0, k, pt, None, None, None, None, pi, pv, *s1) == 0
        assert api.submit_distillation_loss(hdl, 0, dt, n_rows, n_cols, n_cols, n_cols, s, k, px, pi, pv, pw, ploss, pmean, pk, *s3) == 0
        assert api.submit_token_logprobs(hdl, 0, dt, n_rows, n_cols, n_cols, 1.0, 1, 0, px, ptok, plp, pe, pl, None, None, *s2) == 0
        assert api.submit_token_logprobs_bwd(hdl, 0, dt, n_rows, n_cols, n_cols, n_cols, 1.0, 1, px, ptok, pl, pe, pg, ph, pd) == 0
        ids, v = d.get(pi, (n_rows, k), np.uint32), d.get(pv, (n_rows, k), np.float32)
        lse, ent = d.get(pl, (n_rows,), np.float32), d.get(pe, (n_rows,), np.float32)
        w = want_logprobs(dt, t, n_cols, 1.0, tok, k)
        assert np.array_equal(ids, w["top_ids"])
        close(v, w["top_logprobs"], logprob_tol(n_cols, w["top_logprobs"]), "teacher")
        check_distill(dt, x, n_cols, s, ids, v, wt, (d.get(ploss, (n_rows,), np.float32), d.get(pmean, (1,), np.float32), d.get(pk, x.shape, NP_STORAGE[dt])))
        check_logprobs(dt, x, n_cols, 1.0, tok, 0, dict(logprobs=d.get(plp, (n_rows, 1), np.float32), entropy=ent, lse=lse,
                                                        top_ids=np.empty((n_rows, 0), np.uint32), top_logprobs=np.empty((n_rows, 0), np.float32)))
        rounded_once(d.get(pd, x.shape, NP_STORAGE[dt]), dt, want_grad(dt, x, n_cols, 1.0, tok, lse, ent, g, he),
                     grad_slack(dt, x, n_cols, 1.0, tok, lse, ent, g, he), "dlogits")


def test_repeated_calls_give_the_same_bits(hdl):
    for n_rows, n_cols, k in ((2, 128256, 100), (300, 5000, 20)):
        x, tok = logits(60, (n_rows, n_cols), n_cols, BF16), tokens_for(61, n_rows, n_cols, 2)
        ids, v = teacher_for(62, n_rows, n_cols, k)
        runs = [run_logprobs(hdl, BF16, x, n_cols, 0.7, tok, k) for _ in range(3)]
        kd = [run_distill(hdl, BF16, x, n_cols, 0.7, ids, v, None) for _ in range(3)]
        for r in runs[1:]:
            assert all(np.array_equal(r[n], runs[0][n]) for n in r)
        for r in kd[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(r, kd[0]))


def test_two_streams_and_two_threads(hdl):
    """calls on two streams from two threads, each with its own buffers and
    workspace, none waiting for the other's"""
    cases = [(2, 128256, 100), (40, 50257, 20)]
    want, got, wrong = {}, {}, []

    def work(i):
        n_rows, n_cols, k = cases[i]
        x, tok = logits(70 + i, (n_rows, n_cols), n_cols, BF16), tokens_for(72, n_rows, n_cols, 1)
        ids, v = teacher_for(73, n_rows, n_cols, k)
        try:
            for _ in range(6):
                got[i] = run_logprobs(hdl, BF16, x, n_cols, 1.0, tok, k, stream=i), run_distill(hdl, BF16, x, n_cols, 1.0, ids, v, None, stream=i)
                if i not in want:
                    want[i] = check_logprobs(BF16, x, n_cols, 1.0, tok, k, got[i][0])
                    check_distill(BF16, x, n_cols, 1.0, ids, v, None, got[i][1])
                    want[i] = got[i]
                if not all(np.array_equal(got[i][0][n], want[i][0][n]) for n in got[i][0]) or not all(np.array_equal(a, b) for a, b in zip(got[i][1], want[i][1])):
                    wrong.append(i)
        except BaseException as e:  # noqa: BLE001 - reported by the test's own thread
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


class Graph:
    """What `calls` submits to stream 0 of the handle, captured into a graph."""

    def __init__(self, h, calls):
        L, self.stream = api.lib(), ctypes.c_void_p(h.stream(0))   # the HIP runtime that the library is linked with
        self.L, self.graph, self.exec = L, ctypes.c_void_p(), ctypes.c_void_p()
        assert L.hipStreamBeginCapture(self.stream, 1) == 0    # thread-local
        try:
            calls()
        finally:
            assert L.hipStreamEndCapture(self.stream, ctypes.byref(self.graph)) == 0
        assert L.hipGraphInstantiate(ctypes.byref(self.exec), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def replay(self):
        assert self.L.hipGraphLaunch(self.exec, self.stream) == 0

    def destroy(self):
        assert self.L.hipGraphExecDestroy(self.exec) == 0 and self.L.hipGraphDestroy(self.graph) == 0


@pytest.mark.parametrize("shape", [(3, 100001, 50), (400, 2000, 10)], ids=lambda s: "%dx%d_k%d" % s)
def test_captured_and_replayed(hdl, shape):
    """a graph of the three ops, replayed on new logits with eager calls of the
    same ops in between: every replay equals the eager result"""
    n_rows, n_cols, k = shape
    x0 = logits(80, (n_rows, n_cols), n_cols, BF16)
    tok, ids = tokens_for(81, n_rows, n_cols, 2), teacher_for(82, n_rows, n_cols, k)
    g, he = normal_f32(83, (n_rows, 2)), normal_f32(84, (n_rows,))
    sizes = (8 * n_rows, 4 * n_rows, 4 * n_rows, 4 * n_rows * k, 4 * n_rows * k, x0.nbytes, 4 * n_rows, 4, x0.nbytes)
    with Dev(hdl) as d:
        px, ptok, pids, pv, pg, ph = d.put(x0), d.put(tok), d.put(ids[0]), d.put(ids[1]), d.put(g), d.put(he)

        def outputs():
            return [d.put(np.zeros(n, np.uint8)) for n in sizes], \
                [space(d, f(BF16, n_rows, n_cols, k)) for f in (api.token_logprobs_workspace, api.distillation_loss_workspace)]

        def calls(o, sp):
            assert api.submit_token_logprobs(hdl, 0, BF16, n_rows, n_cols, n_cols, 1.0, 2, k, px, ptok, o[0], o[1], o[2], o[3], o[4], *sp[0]) == 0
            assert api.submit_token_logprobs_bwd(hdl, 0, BF16, n_rows, n_cols, n_cols, n_cols, 1.0, 2, px, ptok, o[2], o[1], pg, ph, o[5]) == 0
            assert api.submit_distillation_loss(hdl, 0, BF16, n_rows, n_cols, n_cols, n_cols, 0.5, k, px, pids, pv, None, o[6], o[7], o[8], *sp[1]) == 0

        replayed, eager = outputs(), outputs()
        calls(*eager)
        hdl.sync()
        graph = Graph(hdl, lambda: calls(*replayed))
        for i in range(4):
            hdl.to_device(logits(90 + i, (n_rows, n_cols), n_cols, BF16), px)
            graph.replay()
            hdl.sync()
            calls(*eager)
            hdl.sync()
            for a, b, n in zip(replayed[0], eager[0], sizes):
                assert np.array_equal(d.get(a, (n,), np.uint8), d.get(b, (n,), np.uint8)), "replay %d" % i
        graph.destroy()


# each of the kernels that hold rows, with several rows to a workgroup: a wave,
# a few waves, 16 waves
WALKED = [(9001, 301, 0, 7), (800, 40001, 3, 30), (600, 66000, 0, 64), (530, 140003, 5, 20)]


@pytest.mark.parametrize("dt", [BF16, FP16], ids=dt_id)
@pytest.mark.parametrize("shape", WALKED, ids=lambda s: "%dx%d+%d_k%d" % s)
def test_distillation_walks_rows(hdl, dt, shape):
    """workgroups that take several rows: the next row's logits, teacher and
    weight arrive while a row leaves; rows without weight and rows without an
    entry lie between the others"""
    n_rows, n_cols, pad, k = shape
    x = logits(n_cols, (n_rows, n_cols), n_cols + pad, dt)
    ids, v = teacher_for(n_rows, n_rows, n_cols, k)
    wt = np.where(rng(3).random(n_rows) < 0.2, 0.0, rng(4).uniform(0.1, 2.0, n_rows)).astype(np.float32)
    ids[5::97] = NO_TOKEN
    check_distill(dt, x, n_cols, 0.5, ids, v, wt, run_distill(hdl, dt, x, n_cols, 0.5, ids, v, wt))


def test_more_rows_than_workgroups(hdl):
    """1.2 million short rows"""
    n_rows, n_cols, k, m = 1200003, 8, 2, 1
    x = np.tile(logits(110, (3001, n_cols), n_cols, FP32), (400, 1))[:n_rows]
    x = np.ascontiguousarray(np.resize(x, (n_rows, n_cols)))
    tok = np.resize(tokens_for(111, 3001, n_cols, m), (n_rows, m))
    got = run_logprobs(hdl, FP32, x, n_cols, 1.0, tok, k)
    check_logprobs(FP32, x, n_cols, 1.0, tok, k, got)
    g, he = normal_f32(112, (n_rows, m)), normal_f32(113, (n_rows,))
    out = run_grad(hdl, FP32, x, n_cols, 1.0, tok, got["lse"], got["entropy"], g, he)
    rounded_once(out, FP32, want_grad(FP32, x, n_cols, 1.0, tok, got["lse"], got["entropy"], g, he),
                 grad_slack(FP32, x, n_cols, 1.0, tok, got["lse"], got["entropy"], g, he), "dlogits")
    ids, v = (np.resize(a, (n_rows, 3)) for a in teacher_for(114, 3001, n_cols, 3))
    check_distill(FP32, x, n_cols, 1.0, ids, v, None, run_distill(hdl, FP32, x, n_cols, 1.0, ids, v, None))


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("scale", [1e-6, 1e6])
def test_scales_at_the_limits(hdl, dt, scale):
    """nearly uniform rows, and rows whose largest logit takes everything"""
    n_rows, n_cols, k = 6, 5000, 20
    x = logits(120, (n_rows, n_cols), n_cols, dt)
    tok = tokens_for(121, n_rows, n_cols, 2)
    s32 = float(np.float32(scale))
    got = run_logprobs(hdl, dt, x, n_cols, scale, tok, k)
    w = want_logprobs(dt, x, n_cols, scale, tok, k)
    assert np.array_equal(got["top_ids"], w["top_ids"])
    close(got["logprobs"], w["logprobs"], logprob_tol(n_cols, w["logprobs"]), "logprobs")
    close(got["entropy"], w["entropy"], entropy_tol(n_cols), "entropy")
    ids, v = teacher_for(122, n_rows, n_cols, 5)
    loss, mean, dx = run_distill(hdl, dt, x, n_cols, scale, ids, v, None)
    l, m, d = want_distill(dt, x, n_cols, scale, ids, v, None)
    # differences of logarithms reach s times the logits' spread, about 40
    close(loss, l, distill_loss_tol(n_cols, scale, 5) + np.abs(l) * 16 * U32 + 64.0 * max(s32, 1.0) / s32 ** 2 * 64.0 * U32, "loss")
    rounded_once(dx, dt, d, distill_slack(dt, x, n_cols, scale, ids, None), "dlogits")


def test_a_row_of_more_than_4_gib(hdl):
    """one row of 2^31 - 2^24 bf16 logits, a block of 2^24 again and again: its
    log-sum-exp is the block's and log(127), the largest logits' first
    occurrences come first, and the gradient is the same in every block"""
    block, times, k = 1 << 24, 127, 5
    n_cols = block * times
    x = logits(130, (1, block), block, BF16)
    w = want_logprobs(BF16, x, block, 1.0, np.zeros((1, 1), np.uint32), k)
    order = w["top_ids"][0].astype(np.int64)
    tok = np.array([[n_cols - 1, 3]], np.uint32)
    lse = w["lse"] + np.log(times)
    ids, v = np.array([[n_cols - 2, 7]], np.uint32), np.array([[1.0, 0.5]], np.float32)
    xf = to_f64(x, BF16)[0]
    with Dev(hdl) as d:
        p = d.empty(2 * n_cols)
        ptok, plp, pe, pl, pi, pv = d.put(tok), d.empty(8), d.empty(4), d.empty(4), d.empty(4 * k), d.empty(4 * k)
        pids, pvals, ploss, pg, ph = d.put(ids), d.put(v), d.empty(4), d.put(np.array([[0.5, -2.0]], np.float32)), d.put(np.array([0.25], np.float32))
        s1, s2 = space(d, api.token_logprobs_workspace(BF16, 1, n_cols, k)), space(d, api.distillation_loss_workspace(BF16, 1, n_cols, 2))

        def fill():
            hdl.to_device(x, p)
            for i in range(1, times):
                assert hdl.copy(p + 2 * block * i, p, 2 * block) == 0

        def blocks():
            hdl.sync()
            return [hdl.to_host(p + 2 * block * i, (block,), np.uint16) for i in (0, 63, times - 1)]

        fill()
        assert api.submit_token_logprobs(hdl, 0, BF16, 1, n_cols, n_cols, 1.0, 2, k, p, ptok, plp, pe, pl, pi, pv, *s1) == 0
        # per-thread sums of 2^19 and more terms: the depth of the sums is that of the longest thread
        slack = 2.0 ** 20 * U32
        got_l, got_e = d.get(pl, (1,), np.float32), d.get(pe, (1,), np.float32)
        close(got_l, lse, slack, "lse")
        close(got_e, w["entropy"] + np.log(times), 20.0 * slack, "entropy")
        close(d.get(plp, (2,), np.float32), xf[[block - 1, 3]] - lse, slack, "logprobs")
        top = np.concatenate([np.arange(times) * block + order[0]])[:k]
        assert np.array_equal(d.get(pi, (k,), np.uint32), top.astype(np.uint32))
        assert api.submit_token_logprobs_bwd(hdl, 0, BF16, 1, n_cols, n_cols, n_cols, 1.0, 2, p, ptok, pl, pe, pg, ph, p) == 0
        lp = xf - float(got_l[0])
        dx = -np.exp(lp) * (-1.5 + 0.25 * (lp + float(got_e[0])))
        first, mid, last = blocks()
        want = dx.copy()
        rounded_once(mid, BF16, want, np.exp(lp) * 64.0 * (4 * np.abs(lp) + 16) * U32, "the middle block")
        at = np.array([3])
        assert np.array_equal(np.delete(first, at), np.delete(mid, at)) and np.array_equal(last[:-1], mid[:-1])
        assert abs(to_f64(last, BF16)[-1] - (dx[-1] + 0.5)) <= 2.0 ** -9 and abs(to_f64(first, BF16)[3] - (dx[3] - 2.0)) <= 2.0 ** -8
        fill()
        assert api.submit_distillation_loss(hdl, 0, BF16, 1, n_cols, n_cols, n_cols, 1.0, 2, p, pids, pvals, None, ploss, None, p, *s2) == 0
        q = np.exp(v[0].astype(np.float64) - 1.0)
        q /= q.sum()
        close(d.get(ploss, (1,), np.float32), [(q * (np.log(q) - (xf[[block - 2, 7]] - lse[0]))).sum()], 2.0 * slack, "loss")
        first, mid, last = blocks()
        pr = np.exp(xf - lse[0])
        rounded_once(mid, BF16, pr, pr * 2.0 * slack, "the middle block")
        assert np.array_equal(np.delete(first, 7), np.delete(mid, 7)) and np.array_equal(np.delete(last, block - 2), np.delete(mid, block - 2))
        assert abs(to_f64(last, BF16)[block - 2] - (pr[block - 2] - q[0])) <= 2.0 ** -9 and abs(to_f64(first, BF16)[7] - (pr[7] - q[1])) <= 2.0 ** -9


def test_a_row_of_all_the_columns_that_an_int_counts(hdl):
    """2^31 - 1 columns that begin an element behind an aligned address: no
    index passes 31 bits, and the element before the row stays"""
    block, times, k = 1 << 24, 128, 3
    n_cols = block * times - 1
    x = logits(140, (1, block), block, BF16)
    w = want_logprobs(BF16, x, block, 1.0, np.zeros((1, 1), np.uint32), k)
    at = int(w["top_ids"][0][0])
    assert at > 0
    xf = to_f64(x, BF16)[0]
    lse = w["lse"] + np.log(times - np.exp(xf[0] - w["lse"]))
    with Dev(hdl) as d:
        p = d.empty(2 * (n_cols + 1))
        hdl.to_device(x, p)
        for i in range(1, times):
            assert hdl.copy(p + 2 * block * i, p, 2 * block) == 0
        row = p + 2
        ptok, plp, pe, pl, pi, pv, pg = d.put(np.array([[n_cols - 1]], np.uint32)), d.empty(4), d.empty(4), d.empty(4), d.empty(4 * k), d.empty(4 * k), d.put(np.ones((1, 1), np.float32))
        s1 = space(d, api.token_logprobs_workspace(BF16, 1, n_cols, k))
        assert api.submit_token_logprobs(hdl, 0, BF16, 1, n_cols, n_cols, 1.0, 1, k, row, ptok, plp, pe, pl, pi, pv, *s1) == 0
        # 2^17 terms a thread, of four roundings each
        slack = 2.0 ** 20 * U32
        got_l = d.get(pl, (1,), np.float32)
        close(got_l, lse, slack, "lse")
        close(d.get(pe, (1,), np.float32), w["entropy"] + np.log(times), 20.0 * slack, "entropy")
        close(d.get(plp, (1,), np.float32), xf[[block - 1]] - lse, slack, "logprobs")
        assert np.array_equal(d.get(pi, (k,), np.uint32), (np.arange(k) * block + at - 1).astype(np.uint32))
        ids, v, ploss = d.put(np.array([[n_cols - 1]], np.uint32)), d.put(np.ones((1, 1), np.float32)), d.empty(4)
        s2 = space(d, api.distillation_loss_workspace(BF16, 1, n_cols, 1))
        # one entry: the loss is minus its log-probability
        assert api.submit_distillation_loss(hdl, 0, BF16, 1, n_cols, n_cols, n_cols, 1.0, 1, row, ids, v, None, ploss, None, None, *s2) == 0
        close(d.get(ploss, (1,), np.float32), lse - xf[block - 1], slack, "loss")
        assert api.submit_token_logprobs_bwd(hdl, 0, BF16, 1, n_cols, n_cols, n_cols, 1.0, 1, row, ptok, pl, None, pg, None, row) == 0
        hdl.sync()
        first, mid, last = [hdl.to_host(p + 2 * block * i, (block,), np.uint16) for i in (0, 64, times - 1)]
        lp = xf - float(got_l[0])
        rounded_once(mid, BF16, -np.exp(lp), np.exp(lp) * 4.0 * (4 * np.abs(lp) + 16) * U32, "the middle block")
        assert np.array_equal(first[1:], mid[1:]) and first[0] == x[0, 0] and np.array_equal(last[:-1], mid[:-1])
        assert abs(to_f64(last, BF16)[-1] - (1.0 - np.exp(lp[-1]))) <= 2.0 ** -8


def test_rows_beyond_4_gib(hdl):
    """row offsets past 32 bits: rows 2 GiB apart in one buffer, each with the
    results of the same row packed"""
    n_rows, n_cols, stride, k = 4, 5000, (1 << 30) + 8, 9
    x = logits(95, (n_rows, n_cols), n_cols, BF16)
    tok = tokens_for(96, n_rows, n_cols, 1)
    ids, v = teacher_for(97, n_rows, n_cols, k)
    packed, kd = run_logprobs(hdl, BF16, x, n_cols, 1.0, tok, k), run_distill(hdl, BF16, x, n_cols, 1.0, ids, v, None, mean=False)
    lse, ent, g = packed["lse"], packed["entropy"], normal_f32(98, (n_rows, 1))
    grad = run_grad(hdl, BF16, x, n_cols, 1.0, tok, lse, ent, g, g[:, 0].copy())
    with Dev(hdl) as d:
        ptok, pids, pv, pl, pe, pg = d.put(tok), d.put(ids), d.put(v), d.put(lse), d.put(ent), d.put(g)
        plp, pi, pt, ploss = d.empty(4 * n_rows), d.empty(4 * n_rows * k), d.empty(4 * n_rows * k), d.empty(4 * n_rows)
        p = d.empty(2 * ((n_rows - 1) * stride + n_cols))
        s1, s2 = space(d, api.token_logprobs_workspace(BF16, n_rows, n_cols, k)), space(d, api.distillation_loss_workspace(BF16, n_rows, n_cols, k))

        def put_rows():
            for r in range(n_rows):
                hdl.to_device(x[r], p + 2 * r * stride)

        def rows():
            return np.stack([d.get(p + 2 * r * stride, (n_cols,), np.uint16) for r in range(n_rows)])

        put_rows()
        assert api.submit_token_logprobs(hdl, 0, BF16, n_rows, n_cols, stride, 1.0, 1, k, p, ptok, plp, None, None, pi, pt, *s1) == 0
        assert np.array_equal(d.get(plp, (n_rows, 1), np.float32), packed["logprobs"]) and np.array_equal(d.get(pi, (n_rows, k), np.uint32), packed["top_ids"])
        assert api.submit_token_logprobs_bwd(hdl, 0, BF16, n_rows, n_cols, stride, stride, 1.0, 1, p, ptok, pl, pe, pg, pg, p) == 0
        assert np.array_equal(rows(), grad)
        put_rows()
        assert api.submit_distillation_loss(hdl, 0, BF16, n_rows, n_cols, stride, stride, 1.0, k, p, pids, pv, None, ploss, None, p, *s2) == 0
        assert np.array_equal(rows(), kd[2]) and np.array_equal(d.get(ploss, (n_rows,), np.float32), kd[0])
