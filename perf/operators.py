"""The operators on a model's logits next to the softmax and the cross-entropy,
as they are timed: log-probabilities of given tokens with entropy and top
alternatives, their gradient, and the distillation loss from a teacher's top
logits with its gradient.

A case is a dict of a `kind` and the kind's sizes:

  logprobs  submit_token_logprobs: `tokens` given tokens a row, the row's
            entropy and log-sum-exp, the `top` likeliest columns
  grad      submit_token_logprobs_bwd: the logits' gradient from those of the
            log-probabilities and (with `entropy`) of the entropy
  distill   submit_distillation_loss: loss against the teacher's `top` logits
            and (with `train`) the logits' gradient

`pad` columns lie between one row's logits and the next one's, as they do where
the output projection is padded. `masked`: a part of the vocabulary is banned
(-inf), as in constrained decoding.
"""
import math

import torch

own = False

TYPES = {"fp32": (3, torch.float32, 4), "fp16": (4, torch.float16, 2), "bf16": (5, torch.bfloat16, 2)}


def listed():
    return [
        # one sequence's decoding step, with the 20 alternatives that a serving interface returns
        dict(name="logprobs_1x128256_top20", kind="logprobs", rows=1, vocab=128256, pad=0, dtype="bf16", temperature=1.0, tokens=1, top=20, masked=False),
        # a serving batch at a sampling temperature, with banned tokens
        dict(name="logprobs_64x128256_top5", kind="logprobs", rows=64, vocab=128256, pad=0, dtype="fp16", temperature=0.7, tokens=1, top=5, masked=True),
        # scoring of prompts: the log-probability of every next token
        dict(name="logprobs_4096x128256", kind="logprobs", rows=4096, vocab=128256, pad=0, dtype="bf16", temperature=1.0, tokens=1, top=0, masked=False),
        # a teacher's pass over a batch: the alternatives that a student is trained on; an odd vocabulary, so rows are not aligned
        dict(name="logprobs_1021x50257_top64", kind="logprobs", rows=1021, vocab=50257, pad=0, dtype="bf16", temperature=2.0, tokens=1, top=64, masked=False),
        # answers of a multiple-choice question scored in fp32, rows padded
        dict(name="logprobs_300x32000_fp32", kind="logprobs", rows=300, vocab=32000, pad=64, dtype="fp32", temperature=1.0, tokens=4, top=10, masked=False),
        # a policy-gradient step with an entropy bonus
        dict(name="grad_2048x128256", kind="grad", rows=2048, vocab=128256, pad=0, dtype="bf16", temperature=1.0, tokens=1, entropy=True),
        # the same at an odd vocabulary without the bonus
        dict(name="grad_509x50257_fp16", kind="grad", rows=509, vocab=50257, pad=0, dtype="fp16", temperature=0.8, tokens=1, entropy=False),
        # a few rows of a small fp32 model, several tokens each
        dict(name="grad_16x32000_fp32", kind="grad", rows=16, vocab=32000, pad=64, dtype="fp32", temperature=1.0, tokens=3, entropy=True),
        # a student's training step (the largest case)
        dict(name="distill_4096x128256", kind="distill", rows=4096, vocab=128256, pad=0, dtype="bf16", temperature=2.0, top=64, train=True),
        # a student with an odd vocabulary
        dict(name="distill_1024x50257_fp16", kind="distill", rows=1024, vocab=50257, pad=0, dtype="fp16", temperature=1.0, top=32, train=True),
        # the loss alone, on held-out text
        dict(name="distill_eval_256x151936", kind="distill", rows=256, vocab=151936, pad=0, dtype="bf16", temperature=4.0, top=128, train=False),
        # a toy student: latency
        dict(name="distill_7x1000_fp32", kind="distill", rows=7, vocab=1000, pad=0, dtype="fp32", temperature=1.0, top=8, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of these ranges; its bytes are at most the largest listed case's."""
    while True:
        v = _log(rng, 500, 200000)
        c = dict(kind=rng.choice(["logprobs", "logprobs", "grad", "distill", "distill"]), rows=_log(rng, 1, 8192),
                 vocab=v | 1 if rng.random() < 0.5 else v & ~7, pad=rng.choice([0, 0, 0, rng.randint(1, 129)]),
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), temperature=rng.choice([1.0, round(rng.uniform(0.5, 5.0), 2)]))
        if c["kind"] == "logprobs":
            c.update(tokens=rng.choice([1, 1, rng.randint(2, 32)]), top=rng.choice([0, rng.randint(1, 20), _log(rng, 21, 128)]), masked=rng.random() < 0.25)
        elif c["kind"] == "grad":
            c.update(tokens=rng.choice([1, 1, rng.randint(2, 32)]), entropy=rng.random() < 0.5)
        else:
            c.update(top=_log(rng, 1, 128), train=rng.random() < 0.75)
        if work(c)["bytes"] <= 2.1e9:
            return c


# ---------------- inputs ----------------

def _logits(case, g):
    """Logits of a trained model: a spread of 2.5, an offset of its own for each
    row, and one column well above the rest. Returns them and that column."""
    rows, width = case["rows"], case["vocab"] + case["pad"]
    x = torch.empty((rows, width), dtype=TYPES[case["dtype"]][1], device="cuda").normal_(0.0, 2.5, generator=g)
    x += torch.randn((rows, 1), generator=g, device="cuda").mul_(2.0).to(x.dtype)
    likely = torch.randint(0, case["vocab"], (rows, 1), generator=g, device="cuda")
    peak = torch.rand((rows, 1), generator=g, device="cuda").mul_(14.0).add_(2.0)
    x.scatter_add_(1, likely, peak.to(x.dtype))
    return x, likely


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, vocab, kind = case["rows"], case["vocab"], case["kind"]
    x, likely = _logits(case, g)
    s = dict(case=case, x=x, scale=1.0 / case["temperature"])
    f32 = dict(dtype=torch.float32, device="cuda")
    if kind == "distill":
        k = case["top"]
        # the teacher's alternatives: distinct columns, the student's likeliest among them for most rows
        start = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
        start = torch.where(torch.rand((rows, 1), generator=g, device="cuda") < 0.75, likely, start)
        step = max(1, vocab // (k + 1))
        ids = (start + torch.arange(k, device="cuda") * step) % vocab
        t = torch.randn((rows, k), generator=g, device="cuda").mul_(1.5)
        t += torch.linspace(6.0, 0.0, k, device="cuda")
        # a list may be shorter than its row: the rest holds no column
        short = torch.randint(0, 4 * k + 1, (rows, 1), generator=g, device="cuda")
        ids = torch.where(torch.arange(k, device="cuda") > short, -1, ids)
        s["ids"], s["values"] = ids.to(torch.int32), t
        # tokens of the prompt do not count
        s["weights"] = (torch.rand((rows,), generator=g, device="cuda") < 0.9).float()
        s["loss"], s["mean"] = torch.empty((rows,), **f32), torch.empty((1,), **f32)
        s["dx"] = torch.empty((rows, vocab), dtype=x.dtype, device="cuda") if case["train"] else None
        return s
    if case.get("masked"):
        banned = torch.rand((vocab,), generator=g, device="cuda") < 0.3
        x[:, :vocab].masked_fill_(banned, -math.inf)
        x.scatter_(1, likely, 12.0)
    tok = torch.randint(0, vocab, (rows, case["tokens"]), generator=g, device="cuda")
    tok[:, :1] = torch.where(torch.rand((rows, 1), generator=g, device="cuda") < 0.75, likely, tok[:, :1])
    s["tokens"] = tok.to(torch.int32)
    if kind == "logprobs":
        s["logprobs"], s["entropy"], s["lse"] = (torch.empty(n, **f32) for n in ((rows, case["tokens"]), (rows,), (rows,)))
        if case["top"]:
            s["top_ids"], s["top_logprobs"] = torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda"), torch.empty((rows, case["top"]), **f32)
        return s
    # what the forward pass left, and the loss's gradients
    z = x[:, :vocab].float().mul_(s["scale"])
    s["lse"] = torch.logsumexp(z, 1)
    z -= s["lse"][:, None]
    s["entropy"] = -(z.exp() * z).sum(1)
    s["dlogprobs"] = torch.randn((rows, case["tokens"]), generator=g, device="cuda")
    s["dentropy"] = torch.rand((rows,), generator=g, device="cuda").mul_(-0.02) if case["entropy"] else None
    s["dx"] = torch.empty((rows, vocab), dtype=x.dtype, device="cuda")
    return s


# ---------------- the framework's operators ----------------

_program = {}


def _handle():
    """The program's one handle and its workspace, which grows to the largest call's."""
    if not _program:
        from dataflow_lib_amd import api
        _program.update(api=api, handle=api.Handle(0, num_streams=2, scores=True), space=torch.empty(0, dtype=torch.uint8, device="cuda"))
    return _program["api"], _program["handle"]


def _space(nbytes):
    if _program["space"].numel() < nbytes:
        torch.cuda.synchronize()
        _program["space"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return nbytes, _program["space"].data_ptr() if nbytes else None


def _call(s):
    """The call as arguments: made on a state's first pass, kept with its buffers."""
    api, hd = _handle()
    c, p = s["case"], lambda n: None if s.get(n) is None else s[n].data_ptr()
    dt, rows, vocab, stride = TYPES[c["dtype"]][0], c["rows"], c["vocab"], s["x"].stride(0)
    if c["kind"] == "logprobs":
        space = _space(api.token_logprobs_workspace(dt, rows, vocab, c["top"]))
        return api.submit_token_logprobs, (hd, 0, dt, rows, vocab, stride, s["scale"], c["tokens"], c["top"], p("x"), p("tokens"), p("logprobs"),
                                           p("entropy"), p("lse"), p("top_ids"), p("top_logprobs"), *space)
    if c["kind"] == "grad":
        return api.submit_token_logprobs_bwd, (hd, 0, dt, rows, vocab, stride, vocab, s["scale"], c["tokens"], p("x"), p("tokens"), p("lse"),
                                               p("entropy"), p("dlogprobs"), p("dentropy"), p("dx"))
    space = _space(api.distillation_loss_workspace(dt, rows, vocab, c["top"]))
    return api.submit_distillation_loss, (hd, 0, dt, rows, vocab, stride, vocab, s["scale"], c["top"], p("x"), p("ids"), p("values"), p("weights"),
                                          p("loss"), p("mean"), p("dx"), *space)


OUTPUTS = {"logprobs": ("logprobs", "entropy", "lse", "top_ids", "top_logprobs"), "grad": ("dx",), "distill": ("loss", "mean", "dx")}


def run(s):
    if not own:
        return PLAIN[s["case"]["kind"]](s)
    if "call" not in s or s["space"] is not _program["space"]:
        s["call"] = _call(s)
        s["space"] = _program["space"]
    submit, args = s["call"]
    if submit(*args) != 0:
        raise RuntimeError("%s failed" % submit.__name__)
    return {n: s[n] for n in OUTPUTS[s["case"]["kind"]] if s.get(n) is not None}


# ---------------- their plain forms ----------------

def _order(x):
    """Whole numbers, no two of a row alike, that lie as a row's values do and,
    where values are equal, the lower column's above."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return (bits << 32) - torch.arange(x.shape[1], device=x.device)


def _plain_logprobs(s):
    c = s["case"]
    x = s["x"][:, :c["vocab"]]
    z = x.float() * s["scale"]
    m = z.amax(1, keepdim=True)
    z = z - m
    e = z.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    out = {"logprobs": z.gather(1, s["tokens"].long()) - log_total, "lse": (m + log_total)[:, 0],
           "entropy": (log_total - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total)[:, 0]}
    if c["top"]:
        top = torch.topk(_order(x), c["top"], dim=1).values
        ids = -top & 0xFFFFFFFF
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), z.gather(1, ids) - log_total
    return out


def _plain_grad(s):
    c, scale = s["case"], s["scale"]
    d = s["x"][:, :c["vocab"]].float() * scale - s["lse"][:, None]
    down = s["dlogprobs"].sum(1, keepdim=True)
    if s["dentropy"] is not None:
        down = down + s["dentropy"][:, None] * (d + s["entropy"][:, None])
    dx = d.exp() * down * -scale
    dx.scatter_add_(1, s["tokens"].long(), s["dlogprobs"] * scale)
    return {"dx": dx.to(s["x"].dtype)}


def _plain_distill(s):
    c, scale = s["case"], s["scale"]
    z = s["x"][:, :c["vocab"]].float() * scale
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    ids, there = s["ids"].long().clamp(min=0), s["ids"] >= 0
    v = torch.where(there, s["values"] * scale, -math.inf)
    v = v - v.amax(1, keepdim=True)
    q = v.exp()
    all_q = q.sum(1, keepdim=True)
    log_q, q = v - all_q.log(), q / all_q
    log_p = z.gather(1, ids) - total.log()
    loss = torch.where(there, q * (log_q - log_p), 0.0).sum(1) / scale ** 2
    out = {"loss": torch.where(s["weights"] != 0, loss, 0.0), "mean": (loss * s["weights"]).sum(0, keepdim=True) / c["rows"]}
    if c["train"]:
        w = s["weights"][:, None] / scale
        dx = e / total * w
        dx.scatter_add_(1, ids, -q * w)
        out["dx"] = dx.to(s["x"].dtype)
    return out


PLAIN = {"logprobs": _plain_logprobs, "grad": _plain_grad, "distill": _plain_distill}


# ---------------- what a pass cannot do without, and its answer in 64 bits ----------------

def work(case):
    rows, e = case["rows"], TYPES[case["dtype"]][2]
    n = rows * case["vocab"]
    if case["kind"] == "logprobs":
        return {"bytes": n * e + rows * (8 * case["tokens"] + 8 + 8 * case["top"]), "flops": 7 * n}
    if case["kind"] == "grad":
        return {"bytes": 2 * n * e + rows * (8 * case["tokens"] + (12 if case["entropy"] else 4)), "flops": (7 if case["entropy"] else 4) * n}
    return {"bytes": (2 if case["train"] else 1) * n * e + rows * (8 * case["top"] + 8), "flops": (8 if case["train"] else 4) * n}


def _exact_rows(case, s, at):
    scale = float(torch.tensor(s["scale"], dtype=torch.float32))
    x = s["x"][at, :case["vocab"]].double()
    if case["kind"] == "grad":
        tok, g = s["tokens"][at].long(), s["dlogprobs"][at].double()
        lp = x * scale - s["lse"][at].double().unsqueeze(1)
        p = torch.exp(lp)
        onehots = torch.zeros_like(p).scatter_add(1, tok, g)
        d = onehots - p * g.sum(1, keepdim=True)
        if s["dentropy"] is not None:
            d -= s["dentropy"][at].double().unsqueeze(1) * p * (lp + s["entropy"][at].double().unsqueeze(1))
        return {"dx": d * scale}
    lp = torch.log_softmax(x * scale, dim=1)
    if case["kind"] == "logprobs":
        out = {"logprobs": lp.gather(1, s["tokens"][at].long()), "lse": torch.logsumexp(x * scale, 1), "entropy": torch.special.entr(lp.exp()).sum(1)}
        if case["top"]:
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), lp.gather(1, ids)
        return out
    here = s["ids"][at] != -1
    ids = s["ids"][at].long() * here
    log_q = torch.log_softmax(torch.where(here, s["values"][at].double() * scale, -math.inf), dim=1)
    q = log_q.exp()
    loss = (q * (log_q - lp.gather(1, ids))).masked_fill(~here, 0.0).sum(1) / scale ** 2
    w = s["weights"][at].double()
    out = {"loss": loss * (w != 0), "mean": loss * w}
    if case["train"]:
        out["dx"] = (lp.exp() - torch.zeros_like(lp).scatter_add(1, ids, q)) * (w / scale).unsqueeze(1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    some = max(1, (1 << 27) // case["vocab"])
    parts = [_exact_rows(case, s, slice(r, r + some)) for r in range(0, case["rows"], some)]
    out = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    if "mean" in out:
        out["mean"] = out["mean"].sum(0, keepdim=True) / case["rows"]
    return out
