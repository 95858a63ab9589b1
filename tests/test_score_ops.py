"""The scoring ops (include/dataflow_score_ops.h) without a GPU: their oracle
against other definitions, registration, the arguments' way through the
handle, and every refusal of the launch configuration."""
import ctypes
import math

import numpy as np
import pytest
from scipy.special import log_softmax, logsumexp

from score_support import (DTS, NO_TOKEN, close, dt_id, logits, logprob_tol, rounded_once, score_oracle, teacher_for, tokens_for, want_distill, want_grad,
                           want_logprobs)
from support import BF16, FP32, ORACLE_LIB, normal, ptr, rng, to_f64

from dataflow_lib_amd import api

OPS = ["token_logprobs", "token_logprobs_bwd", "distillation_loss"]
NUM_ARGS = {"token_logprobs": 15, "token_logprobs_bwd": 13, "distillation_loss": 15}


# ---------------- the oracle ----------------

@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("scale", [1.0, 0.5, 2.5])
def test_oracle_logprobs_against_scipy(dt, scale):
    x = logits(1, (6, 301), 305, dt)
    tok = tokens_for(2, 6, 301, 3)
    w = want_logprobs(dt, x, 301, scale, tok, 7)
    xf = to_f64(x, dt)[:, :301]
    lp = log_softmax(scale * xf, axis=1)
    assert np.allclose(w["lse"], logsumexp(scale * xf, axis=1), rtol=1e-13, atol=1e-13)
    assert np.allclose(w["entropy"], -(np.exp(lp) * lp).sum(1), rtol=1e-12)
    there = tok < 301
    assert np.allclose(w["logprobs"][there], np.take_along_axis(lp, np.where(there, tok, 0).astype(int), 1)[there], rtol=1e-13)
    assert np.all(w["logprobs"][~there] == 0.0) and (~there).sum() == 2
    order = np.argsort(-xf, axis=1, kind="stable")[:, :7]
    assert np.array_equal(w["top_ids"], order) and np.allclose(w["top_logprobs"], np.take_along_axis(lp, order, 1), rtol=1e-13)


def test_oracle_odd_rows():
    x = np.array([[1.0, 1.0, 0.0, 1.0], [-np.inf] * 4, [0.0, -np.inf, -0.0, -1.0], [np.nan, 2.0, -np.inf, 3.0], [np.finfo(np.float32).min] * 4,
                  [np.inf, 0.0, 0.0, 0.0]], np.float32)
    w = want_logprobs(FP32, x, 4, 1.0, np.array([[0], [1], [1], [1], [3], [1]], np.uint32), 4)
    assert w["top_ids"].tolist() == [[0, 1, 3, 2], [0, 1, 2, 3], [0, 2, 3, 1], [3, 1, 2, 0], [0, 1, 2, 3], [0, 1, 2, 3]]
    assert w["lse"][1] == -np.inf and w["entropy"][1] == 0.0 and w["logprobs"][1, 0] == -np.inf
    assert w["logprobs"][2, 0] == -np.inf and math.isclose(w["logprobs"][4, 0], -math.log(4.0)) and math.isclose(w["entropy"][4], math.log(4.0))
    assert np.isnan(w["lse"][[3, 5]]).all() and np.isnan(w["entropy"][[3, 5]]).all()


def numeric(f, x, h=1e-5):
    g = np.empty_like(x)
    for j in range(x.size):
        a, b = x.copy(), x.copy()
        a[j] += h
        b[j] -= h
        g[j] = (f(a) - f(b)) / (2 * h)
    return g


def test_oracle_gradients_against_differences():
    """dlogits of sum g logprob + h entropy, and of w * distillation loss, with
    tokens given twice and tokens that are no column"""
    n, s = 23, 0.7
    s32 = float(np.float32(s))
    x = logits(3, (2, n), n, FP32)
    tok = np.array([[3, 3, 22, NO_TOKEN], [0, 5, n, 1]], np.uint32)
    g, h = normal(4, (2, 4)), normal(5, (2,))
    w = want_logprobs(FP32, x, n, s, tok, 0)
    dx = want_grad(FP32, x, n, s, tok, w["lse"].astype(np.float32), w["entropy"].astype(np.float32), g, h)
    ids = np.array([[3, 3, 22, NO_TOKEN], [0, 5, 7, 1]], np.uint32)
    v, wt = np.array([[1.0, 0.5, 2.0, 9.0], [0.1, -np.inf, 0.3, 0.2]], np.float32), np.array([0.5, 2.0], np.float32)
    loss, mean, dk = want_distill(FP32, x, n, s, ids, v, wt)
    assert np.isclose(mean[0], (loss * wt).sum() / 2, rtol=1e-14)
    for r in range(2):
        def policy(z):
            lp = log_softmax(s32 * z)
            return sum(g[r, m] * lp[t] for m, t in enumerate(tok[r]) if t < n) - h[r] * (np.exp(lp) * lp).sum()

        def kd(z):
            lp = log_softmax(s32 * z)
            keep = [k for k in range(4) if ids[r, k] < n and np.isfinite(v[r, k])]
            lq = log_softmax(s32 * v[r, keep].astype(np.float64))
            return sum(np.exp(a) * (a - lp[ids[r, k]]) for a, k in zip(lq, keep)) / s32 ** 2

        row = x[r].astype(np.float64)
        assert np.allclose(dx[r], numeric(policy, row), rtol=1e-5, atol=1e-6)   # lse and entropy are given in fp32
        assert math.isclose(loss[r], kd(row), rel_tol=1e-12)
        assert np.allclose(dk[r], wt[r] * numeric(kd, row), rtol=1e-7, atol=1e-9)


def test_oracle_distillation_closed_forms():
    """a teacher that is the student over all columns: no loss, no gradient;
    one entry: the cross-entropy of that column"""
    n = 9
    x = logits(6, (1, n), n, FP32)
    ids = np.arange(n, dtype=np.uint32)[None]
    loss, _, dx = want_distill(FP32, x, n, 0.5, ids, x.copy(), None)
    assert abs(loss[0]) < 1e-14 and np.abs(dx).max() < 1e-14
    loss, _, dx = want_distill(FP32, x, n, 1.0, np.array([[4]], np.uint32), np.array([[7.0]], np.float32), None)
    lp = log_softmax(x[0].astype(np.float64))
    assert math.isclose(loss[0], -lp[4], rel_tol=1e-14) and np.allclose(dx[0], np.exp(lp) - np.eye(n)[4], atol=1e-15)


def test_tolerances_reject_lost_precision():
    """a sum of exponentials in bf16, and a gradient rounded twice, fail"""
    x = logits(7, (4, 4096), 4096, BF16)
    xf = to_f64(x, BF16)
    z = (xf - xf.max(1, keepdims=True))
    lz = np.log(np.exp(z).sum(1))
    bad = np.log(to_f64(np.asarray((np.exp(z).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)), BF16).sum(1))
    with pytest.raises(AssertionError):
        close(z[:, 0] - bad, z[:, 0] - lz, logprob_tol(4096, z[:, 0] - lz), "truncated terms")
    v = np.full(8, 1.0 + 2.0 ** -8 + 2.0 ** -12)
    rounded_once(np.full(8, 0x3F81, np.uint16), BF16, v, 0.0, "nearest")
    with pytest.raises(AssertionError):
        rounded_once(np.full(8, 0x3F80, np.uint16), BF16, v, 0.0, "the other neighbour")


# ---------------- registration and marshalling ----------------

@pytest.fixture(scope="module")
def cpu_handle():
    O = score_oracle()
    O.init_cpu_dataflow_handle.argtypes = [ctypes.POINTER(api.DataflowHandle), ctypes.c_int]
    O.destroy_cpu_dataflow_handle.argtypes = [ctypes.POINTER(api.DataflowHandle)]
    h = api.DataflowHandle()
    assert O.init_cpu_dataflow_handle(ctypes.byref(h), 1) == 0
    assert api.lib().register_native_ops(ctypes.byref(h), ORACLE_LIB.encode(), b"") == 68
    assert api.lib().register_native_score_ops(ctypes.byref(h), ORACLE_LIB.encode(), b"") == 9
    yield h
    O.destroy_cpu_dataflow_handle(ctypes.byref(h))


def test_registration_adds_the_nine_functions(cpu_handle):
    assert cpu_handle.num_ops == 77 and cpu_handle.op_table.cnt == 77


@pytest.mark.parametrize("op", OPS)
def test_skeletons(op):
    seen = set()
    for dt in DTS:
        sk = api.native_op_skeleton(op, dt)
        assert sk.header.op_nickname.decode() == "%s_%s" % (op, api.datatype_as_string(dt)) and sk.header.num_args == NUM_ARGS[op]
        seen.add(bytes(sk.fingerprint))
        own = api.OpSkeleton()
        getattr(api.lib(), "set_native_%s_skeleton" % op)(ctypes.byref(own), dt)
        assert bytes(own) == bytes(sk)
    assert len(seen) == 3


def test_unregistered_types_are_refused(cpu_handle):
    x = np.zeros((1, 8), np.float32)
    assert api.submit_token_logprobs(ctypes.byref(cpu_handle), 0, api.DATAFLOW_FP8E4M3, 1, 8, 8, 1.0, 0, 0, ptr(x), None, None, None, None, None, None) == -1


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
def test_arguments_through_the_handle(cpu_handle, dt):
    """the three ops as they are used together: a teacher's alternatives become
    the student's distillation targets; row and gradient strides differ"""
    H = ctypes.byref(cpu_handle)
    R, n, stride, gstride, M, K, s = 5, 40, 43, 47, 3, 6, 0.5
    x, tok = logits(8, (R, n), stride, dt), tokens_for(9, R, n, M)
    f = lambda *sh: np.full(sh, 7.0, np.float32)  # noqa: E731
    lp, ent, lse, tid, tlp = f(R, M), f(R), f(R), np.zeros((R, K), np.uint32), f(R, K)
    assert api.submit_token_logprobs(H, 0, dt, R, n, stride, s, M, K, ptr(x), ptr(tok), ptr(lp), ptr(ent), ptr(lse), ptr(tid), ptr(tlp)) == 0
    w = want_logprobs(dt, x, n, s, tok, K)
    for got, name in ((lp, "logprobs"), (ent, "entropy"), (lse, "lse"), (tid, "top_ids"), (tlp, "top_logprobs")):
        assert np.array_equal(got, w[name].astype(got.dtype)), name
    g, h = normal(10, (R, M)), normal(11, (R,))
    blank = to_storage_like(dt, (R, gstride))
    dx = blank.copy()
    assert api.submit_token_logprobs_bwd(H, 0, dt, R, n, stride, gstride, s, M, ptr(x), ptr(tok), ptr(lse), ptr(ent), ptr(g), ptr(h), ptr(dx)) == 0
    rounded_once(dx[:, :n], dt, want_grad(dt, x, n, s, tok, lse, ent, g, h), 1e-30, "dlogits")
    assert np.array_equal(dx[:, n:], blank[:, n:])
    y, wt = logits(12, (R, n), stride, dt), np.array([1, 0, 2, 1, 0.5], np.float32)
    loss, mean, dy = f(R), f(1), blank.copy()
    assert api.submit_distillation_loss(H, 0, dt, R, n, stride, gstride, s, K, ptr(y), ptr(tid), ptr(tlp), ptr(wt), ptr(loss), ptr(mean), ptr(dy)) == 0
    l, m, d = want_distill(dt, y, n, s, tid, tlp, wt)
    assert np.array_equal(loss, l.astype(np.float32)) and loss[1] == 0.0 and mean[0] == np.float32(m[0])
    rounded_once(dy[:, :n], dt, d, 1e-30, "distillation dlogits")
    assert np.array_equal(dy[:, n:], blank[:, n:]) and not to_f64(dy, dt)[1, :n].any()


def to_storage_like(dt, shape):
    from support import to_storage
    return to_storage(np.full(shape, 3.0, np.float32), dt)


# ---------------- refusals ----------------

class HipFunction(ctypes.Structure):
    """Hip_Function (hip_dataflow_handle.h)"""
    _fields_ = [("func_max_smem", ctypes.c_int), ("func_max_threads_per_block", ctypes.c_int), ("shares_module_scratch", ctypes.c_int),
                ("occupancy_memo", ctypes.c_uint64 * 9), ("is_native", ctypes.c_bool), ("function_handle", ctypes.c_void_p),
                ("set_launch_config", ctypes.c_void_p), ("finish_function_handle", ctypes.c_void_p), ("variant_handles", ctypes.c_void_p * 8),
                ("set_finish_launch_config", ctypes.c_void_p), ("hip_external_func", ctypes.c_void_p), ("op_extra", ctypes.c_void_p),
                ("op_skeleton", api.OpSkeleton)]


class LaunchConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint) for n in ("gridDimX", "gridDimY", "gridDimZ", "blockDimX", "blockDimY", "blockDimZ", "sharedMemBytes",
                                             "variant", "then_variant")]


I, U, F, P = ctypes.c_int, ctypes.c_uint64, ctypes.c_float, ctypes.c_void_p
ARGS = {
    "token_logprobs": [("n_rows", I), ("n_cols", I), ("row_stride", U), ("scale", F), ("tokens_per_row", I), ("top_k", I), ("logits", P), ("tokens", P),
                       ("logprobs", P), ("entropy", P), ("lse", P), ("top_ids", P), ("top_logprobs", P), ("workspaceBytes", U), ("workspace", P)],
    "token_logprobs_bwd": [("n_rows", I), ("n_cols", I), ("row_stride", U), ("grad_stride", U), ("scale", F), ("tokens_per_row", I), ("logits", P),
                           ("tokens", P), ("lse", P), ("entropy", P), ("d_logprobs", P), ("d_entropy", P), ("dlogits", P)],
    "distillation_loss": [("n_rows", I), ("n_cols", I), ("row_stride", U), ("grad_stride", U), ("scale", F), ("top_k", I), ("logits", P),
                          ("teacher_ids", P), ("teacher_logits", P), ("row_weights", P), ("loss", P), ("mean_loss", P), ("dlogits", P),
                          ("workspaceBytes", U), ("workspace", P)],
}
# a call that is accepted: 4 rows of 100 columns; pointers are never followed
GOOD = dict(n_rows=4, n_cols=100, row_stride=104, grad_stride=108, scale=1.0, tokens_per_row=2, top_k=5, logits=0x100000, dlogits=0x200000,
            workspaceBytes=1 << 40, workspace=0x40000000,
            **{n: 0x300000 for n in ("tokens", "logprobs", "entropy", "lse", "top_ids", "top_logprobs", "d_logprobs", "d_entropy", "teacher_ids",
                                     "teacher_logits", "row_weights", "loss", "mean_loss")})


def config(op, dt=BF16, finish=False, **change):
    """(status, launch configuration) of a call that differs from GOOD"""
    lib = ctypes.CDLL(api.CONFIG_LIB)
    f, c, info, h, o = HipFunction(), LaunchConfig(), api.HipDeviceInfo(), api.DataflowHandle(), api.Op()
    f.op_skeleton = api.native_op_skeleton(op, dt)
    info.cu_count, info.max_smem_per_block = 256, 160 << 10
    h.device_info = ctypes.cast(ctypes.byref(info), ctypes.c_void_p)
    values = {**GOOD, **change}
    held = [t(values[n]) for n, t in ARGS[op]]
    for i, v in enumerate(held):
        o.op_args[i] = ctypes.cast(ctypes.byref(v), ctypes.c_void_p)
    fn = getattr(lib, op + ("_set_finish_launch_config" if finish else "_set_launch_config"))
    return fn(ctypes.byref(c), ctypes.byref(h), ctypes.byref(f), ctypes.byref(o)), c


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("dt", DTS, ids=dt_id)
def test_accepted_calls(op, dt):
    rc, c = config(op, dt)
    assert rc == 0 and c.gridDimX >= 1 and c.blockDimX % 64 == 0 and c.gridDimX * c.blockDimX < 2 ** 32


@pytest.mark.parametrize("op", OPS)
def test_empty_calls_launch_nothing(op):
    for change in (dict(n_rows=0), dict(n_cols=0), dict(n_rows=0, logits=None, dlogits=None)):
        rc, c = config(op, **change)
        assert rc == 0 and c.gridDimX == 0, change


COMMON = [dict(n_rows=-1), dict(n_cols=-1), dict(row_stride=99), dict(row_stride=2 ** 63), dict(row_stride=2 ** 60), dict(scale=0.0), dict(scale=-1.0),
          dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e-7), dict(scale=2e6), dict(logits=None), dict(logits=0x100001)]
REFUSED = {
    "token_logprobs": [dict(tokens_per_row=-1), dict(tokens_per_row=1025), dict(top_k=-1), dict(top_k=257), dict(top_k=101), dict(tokens=None),
                       dict(logprobs=None), dict(top_ids=None), dict(top_logprobs=None), dict(tokens=0x300002), dict(lse=0x300001), dict(entropy=0x300002)],
    "token_logprobs_bwd": [dict(tokens_per_row=-1), dict(tokens_per_row=1025), dict(tokens=None), dict(d_logprobs=None), dict(lse=None),
                           dict(entropy=None), dict(dlogits=None), dict(dlogits=0x200001), dict(grad_stride=99), dict(grad_stride=2 ** 62),
                           dict(dlogits=0x100000), dict(dlogits=0x100002, grad_stride=104), dict(dlogits=0x100000 + 2 * (3 * 104 + 99)),
                           dict(dlogits=0x100000 - 2 * (3 * 108 + 99)), dict(d_entropy=0x300001)],
    "distillation_loss": [dict(top_k=-1), dict(top_k=1025), dict(teacher_ids=None), dict(teacher_logits=None), dict(loss=None), dict(mean_loss=0x300002),
                          dict(row_weights=0x300001), dict(dlogits=0x200001), dict(grad_stride=99), dict(dlogits=0x100000),
                          dict(dlogits=0x100002, grad_stride=104)],
}


@pytest.mark.parametrize("op,change", [(op, c) for op in OPS for c in COMMON + REFUSED[op]], ids=lambda v: v if isinstance(v, str) else str(v))
def test_refused_calls(op, change):
    assert config(op, **change)[0] == -1


@pytest.mark.parametrize("op,change", [
    ("token_logprobs", dict(tokens_per_row=0, tokens=None, logprobs=None)), ("token_logprobs", dict(top_k=0, top_ids=None, top_logprobs=None)),
    ("token_logprobs", dict(entropy=None, lse=None)), ("token_logprobs", dict(top_k=100)), ("token_logprobs", dict(tokens_per_row=1024)),
    ("token_logprobs_bwd", dict(tokens_per_row=0, tokens=None, d_logprobs=None)), ("token_logprobs_bwd", dict(d_entropy=None, entropy=None)),
    ("token_logprobs_bwd", dict(dlogits=0x100000, grad_stride=104)), ("token_logprobs_bwd", dict(dlogits=0x100000 + 2 * (3 * 104 + 100))),
    ("token_logprobs_bwd", dict(dlogits=0x100000 - 2 * (3 * 108 + 100))),
    ("distillation_loss", dict(row_weights=None, mean_loss=None, dlogits=None)), ("distillation_loss", dict(dlogits=0x100000, grad_stride=104)),
    ("distillation_loss", dict(top_k=0, teacher_ids=None, teacher_logits=None)), ("distillation_loss", dict(n_rows=1, dlogits=0x100000)),
], ids=lambda v: v if isinstance(v, str) else str(v))
def test_operands_that_may_be_left_out(op, change):
    assert config(op, **change)[0] == 0


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
@pytest.mark.parametrize("op", ["token_logprobs", "distillation_loss"])
def test_workspaces_are_checked(op, dt):
    """over sizes small and large: exactly the bytes that the size function
    gives are enough, fewer, none or an unaligned place are not"""
    size = getattr(api, op + "_workspace")
    g = rng(13)
    asked = 0
    for _ in range(300):
        rows, cols = int(2 ** g.uniform(0, 20)), int(2 ** g.uniform(8.2, 25))
        k = int(g.integers(0, 257))
        need = size(dt, rows, cols, k)
        call = dict(n_rows=rows, n_cols=cols, top_k=k, row_stride=cols, grad_stride=cols, logits=1 << 40, dlogits=1 << 58)
        assert config(op, dt, workspaceBytes=need, workspace=0x40000000 if need else None, **call)[0] == 0
        if need:
            asked += 1
            assert need <= rows * (32 * 16 + (4 * k if op == "distillation_loss" else 32 * 8 * k))
            for space in ((need - 1, 0x40000000), (need, None), (need, 0x40000010), (0, None)):
                assert config(op, dt, workspaceBytes=space[0], workspace=space[1], **call)[0] == -1
    assert size(dt, 0, 100, 5) == 0 and size(dt, 4, 0, 0) == 0 and size(dt, -1, -1, -1) == 0


def test_largest_launches_stay_below_2_to_32_threads():
    for op in OPS:
        for rows, cols in ((2 ** 31 - 1, 1), (2 ** 31 - 1, 64), (2 ** 26, 1000), (1, 2 ** 31 - 1), (3, 2 ** 31 - 1), (2 ** 24, 2 ** 24)):
            rc, c = config(op, n_rows=rows, n_cols=cols, row_stride=cols, grad_stride=cols, top_k=1, logits=1 << 40, dlogits=1 << 58)
            assert rc == 0 and 0 < c.gridDimX * c.blockDimX < 2 ** 32, (op, rows, cols)


def launched(op, dt, n_rows, n_cols, k, **change):
    """(main kernel, kernel launched after it, finish kernel) of a call, by suffix"""
    suffix = ["", "_rows", "_wide_rows", "_long_rows", "_multi", "_split", "_split_out", "_any_rows", "_top"]
    change = dict(n_rows=n_rows, n_cols=n_cols, top_k=k, row_stride=n_cols, grad_stride=n_cols, logits=1 << 40, dlogits=1 << 50) | change
    rc, c = config(op, dt, **change)
    assert rc == 0
    finish = op != "token_logprobs_bwd" and config(op, dt, finish=True, **change)[1].gridDimX > 0
    return suffix[c.variant], suffix[c.then_variant], "_finish" if finish else ""


@pytest.mark.parametrize("dt", DTS, ids=dt_id)
def test_gpu_tests_reach_every_kernel(dt):
    """one slice and several, with and without alternatives; rows held by each
    of the kernels that hold them, and rows read twice"""
    import test_hip_score_ops as T
    logprobs = {launched("token_logprobs", dt, s[0], s[1], s[5]) for s in T.SHAPES}
    assert logprobs == {("", "", ""), ("", "", "_finish"), ("_top", "", ""), ("_top", "", "_finish")}
    distill = {launched("distillation_loss", dt, s[0], s[1], s[6], mean_loss=None)[:2] for s in T.KD_SHAPES}
    walked = {launched("distillation_loss", dt, s[0], s[1], s[3], mean_loss=None)[:2] for s in T.WALKED}
    held = {("_rows", ""), ("_wide_rows", ""), ("_long_rows", ""), ("_any_rows", "")}
    assert distill | walked >= held | {("", "_split_out")} and (dt == FP32 or walked == held)
    alone = {launched("distillation_loss", dt, s[0], s[1], s[6], mean_loss=None, dlogits=None)[:2] for s in T.KD_SHAPES}
    assert alone == {("", ""), ("", "_split_out")}


def test_mean_loss_runs_only_where_it_is_wanted():
    assert config("distillation_loss", finish=True, mean_loss=None)[1].gridDimX == 0
    assert config("distillation_loss", finish=True)[1].gridDimX == 1
