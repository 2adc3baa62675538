"""Cases for the operators that fit a draft head to the target: the lm_head's softmax cross
entropy and its distillation from the target's top logits, forward and backward, and the
top-K of a verify sweep's logits that the distillation reads.

``run`` computes a case in its plain form (fp32 torch operations over written logits), or,
with ``own`` set, through the library's entry points.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

LARGEST = 6.0 * 2048 * 163840 * 7168       # flops of the largest listed case


def _k3():
    if "k3b200" not in sys.modules:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location(
            "k3b200", os.path.join(here, "kimi-k3-for-me_b200", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["k3b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["k3b200"]


# ------------------------------------------------------------------------------ cases --
def _topk(rows, vocab, k, **kw):
    return {"op": "topk", "rows": rows, "vocab": vocab, "k": k, **kw}


def _xent(rows, hidden, vocab, grad, masked=0.0, **kw):
    return {"op": "xent", "rows": rows, "hidden": hidden, "vocab": vocab, "grad": grad, "masked": masked, **kw}


def _distill(rows, hidden, vocab, k, grad, temp=1.0, masked=0.0, **kw):
    return {"op": "distill", "rows": rows, "hidden": hidden, "vocab": vocab, "k": k, "grad": grad, "temp": temp,
            "masked": masked, **kw}


def listed():
    return [
        # the teacher's side of one sequence's sweep: a pending token and 8 drafts
        _topk(9, 163840, 64, name="topk, one sweep"),
        # the same for 64 sequences at once
        _topk(576, 163840, 32, name="topk, 64 sequences"),
        # a draft model's odd vocabulary, few entries kept
        _topk(77, 50257, 10, name="topk, odd vocabulary"),
        # the loss of one short sequence under the full head (scoring, perplexity): a weight stream
        _xent(9, 7168, 163840, "none", name="xent loss, one sweep"),
        # the loss of a validation batch
        _xent(2048, 7168, 163840, "none", masked=0.25, name="xent loss, batch"),
        # a small draft model's training step: latency counts
        _xent(64, 1024, 32000, "both", name="xent step, small"),
        # odd sizes everywhere, a third of the rows prompt tokens without a loss
        _xent(301, 1000, 50257, "both", masked=0.33, name="xent step, odd"),
        # a draft head of its own width over the target's vocabulary
        _xent(4096, 2048, 163840, "both", masked=0.1, name="xent step, draft head"),
        # the target's own head trained at full width: the largest
        _xent(2048, 7168, 163840, "both", name="xent step, full head"),
        # the distillation loss of 64 sequences' sweeps
        _distill(576, 7168, 163840, 64, "none", name="distill loss, 64 sequences"),
        # a drafter that shares the target's frozen head: only the hidden states learn
        _distill(576, 7168, 163840, 32, "x", temp=2.0, name="distill step, frozen head"),
        # a draft head of its own, distilled
        _distill(2048, 2048, 163840, 64, "both", masked=0.1, name="distill step, draft head"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["topk", "xent", "xent", "distill", "distill"])
        vocab = rng.choice([_log(rng, 1000, 163840), _log(rng, 1000, 163840), 32000, 163840])
        if op == "topk":
            return _topk(_log(rng, 1, 576), vocab, _log(rng, 1, 128))
        rows, hidden = _log(rng, 1, 4096), 8 * _log(rng, 8, 896)
        grad = rng.choice(["none", "both", "x"])
        masked = rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.9), 2)])
        if op == "xent":
            case = _xent(rows, hidden, vocab, grad, masked)
        else:
            temp = rng.choice([1.0, 1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)])
            case = _distill(rows, hidden, vocab, _log(rng, 1, 128), grad, temp, masked)
        if work(case)["flops"] <= LARGEST:
            return case


# ------------------------------------------------------------------------------ inputs -
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    if case["op"] == "topk":
        # logits around zero with a confident head per row, a few ids banned (-inf)
        logits = randn(rows, vocab) * 1.7
        hot = torch.randint(0, vocab, (rows, 8), generator=gen, device="cuda")
        logits.scatter_add_(1, hot, randn(rows, 8).abs() * 6.0)
        ban = torch.randint(0, vocab, (max(1, vocab // 1000),), generator=gen, device="cuda")
        logits[:, ban] = -math.inf
        return {"case": dict(case), "logits": logits}

    hidden = case["hidden"]
    # a head whose random logits spread by 1.7, and hidden states after the final norm that
    # lean towards the rows of what comes next, from not at all to confidently
    W = (randn(vocab, hidden, dtype=torch.bfloat16) * (1.7 / math.sqrt(hidden)))
    lean = torch.rand((rows, 1), generator=gen, device="cuda") * 8.0
    keep = torch.rand(rows, generator=gen, device="cuda") >= case["masked"]
    # each row's weight in the batch's mean
    g = keep.float() / keep.sum().clamp(min=1)
    state = {"case": dict(case), "W": W, "g": g}
    if case["op"] == "xent":
        label = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        state["X"] = (randn(rows, hidden) + lean * W[label].float() / 1.7).bfloat16()
        state["label"] = torch.where(keep, label, -100).int()
    else:
        k = case["k"]
        ids = torch.randint(0, vocab, (rows, k), generator=gen, device="cuda")
        gaps = -torch.log(torch.rand((rows, k), generator=gen, device="cuda").clamp(min=1e-6)) * (8.0 / (4 + k))
        state["top"] = 18.0 - gaps.cumsum(1)
        state["X"] = (randn(rows, hidden) + lean * W[ids[:, 0]].float() / 1.7).bfloat16()
        state["ids"] = torch.where(keep[:, None], ids, -1).int()
    return state


# --------------------------------------------------------------------------------- run -
def _run_own(s):
    k3, c = _k3(), s["case"]
    if c["op"] == "topk":
        idx, val = k3.topk_logits(s["logits"], c["k"])
        return {"idx": idx, "val": val}
    if c["op"] == "xent":
        loss, lse = k3.lm_head_xent(s["X"], s["W"], s["label"])
    else:
        loss, lse = k3.lm_head_distill(s["X"], s["W"], s["ids"], s["top"], temp=c["temp"])
    out = {"loss": loss, "lse": lse}
    if c["grad"] != "none":
        both = c["grad"] == "both"
        if c["op"] == "xent":
            dx, dw = k3.lm_head_xent_grad(s["X"], s["W"], s["label"], lse, g=s["g"], need_dw=both)
        else:
            dx, dw = k3.lm_head_distill_grad(s["X"], s["W"], s["ids"], s["top"], lse, temp=c["temp"], g=s["g"],
                                             need_dw=both)
        out["dx"] = dx
        if both:
            out["dw"] = dw
    return out


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "topk":
        val, idx = torch.sort(state["logits"], dim=1, descending=True, stable=True)
        return {"idx": idx[:, :c["k"]].int(), "val": val[:, :c["k"]].contiguous()}
    x, w = state["X"].float(), state["W"].float()
    # a row without a target has a loss, an lse and a gradient of zero
    if c["op"] == "xent":
        temp, live = 1.0, state["label"] >= 0
        ids = state["label"].long().clamp(min=0)[:, None]
        q = torch.ones_like(ids, dtype=torch.float32)
        entropy = torch.zeros_like(live, dtype=torch.float32)
    else:
        temp, live = c["temp"], (state["ids"] >= 0).any(1)
        ids = state["ids"].long().clamp(min=0)
        t = (state["top"] - state["top"].amax(1, keepdim=True)) / temp
        q = torch.exp(t)
        total = q.sum(1, keepdim=True)
        q = q / total
        entropy = (q * (t - torch.log(total))).sum(1)
    z = (x @ w.t()) / temp
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    loss = entropy + (q * (lse - z.gather(1, ids))).sum(1)
    zero = torch.zeros_like(loss)
    out = {"loss": torch.where(live, loss, zero), "lse": torch.where(live, lse[:, 0], zero)}
    if c["grad"] != "none":
        dz = torch.exp(z - lse).scatter_add_(1, ids, -q)
        dz = dz * torch.where(live, state["g"] / temp, zero)[:, None]
        out["dx"] = (dz @ w).bfloat16()
        if c["grad"] == "both":
            out["dw"] = (dz.t() @ x).bfloat16()
    return out


# -------------------------------------------------------------------------------- work -
def work(case):
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "topk":
        return {"bytes": rows * vocab * 4.0 + rows * case["k"] * 8.0, "flops": float(rows * vocab)}
    live, hidden = rows * (1.0 - case["masked"]), case["hidden"]
    size, head = live * hidden * 2.0, vocab * hidden * 2.0
    product = 2.0 * live * vocab * hidden
    grads = {"none": 0, "x": 1, "both": 2}[case["grad"]]
    targets = rows * (case["k"] * 8.0 if case["op"] == "distill" else 4.0)
    return {"bytes": size + head + targets + rows * 8.0 + (size if grads else 0.0) + (head if grads == 2 else 0.0),
            "flops": product * (1 + grads)}


# ------------------------------------------------------------------------------- exact -
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "topk":
        # one whole number a value, ordered as (value, lowest id first)
        bits = s["logits"].view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        span = case["vocab"]
        best = torch.topk(order * span + (span - 1 - torch.arange(span, device="cuda")), case["k"], dim=1).values
        idx = span - 1 - best.remainder(span)
        return {"idx": idx.int(), "val": s["logits"].gather(1, idx).double()}
    rows, grad = case["rows"], case["grad"]
    temp = case.get("temp", 1.0)
    W = s["W"].double()
    X = s["X"].double()
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    lse, dX = torch.zeros_like(loss), torch.zeros_like(X)
    dW = torch.zeros_like(W) if grad == "both" else None
    block = 512
    for r in range(0, rows, block):
        x = X[r:r + block]
        logp = torch.log_softmax(torch.matmul(x, W.T).div_(temp), dim=1)
        target = torch.zeros_like(logp)
        if case["op"] == "xent":
            label = s["label"][r:r + block].long()
            on = label.ge(0)
            target[on, label[on]] = 1.0
            negative_entropy = 0.0
        else:
            ids = s["ids"][r:r + block].long()
            on = ids[:, 0].ge(0)
            logq = torch.log_softmax(s["top"][r:r + block].double() / temp, dim=1)
            negative_entropy = logq.exp().mul(logq).sum(1)
            target.index_put_((torch.arange(len(x), device="cuda")[on][:, None].expand(-1, case["k"]), ids[on]),
                              logq.exp()[on], accumulate=True)
        loss[r:r + block] = (negative_entropy - target.mul(logp).sum(1)) * on
        first = torch.matmul(x, W[0]) / temp
        lse[r:r + block] = (first - logp[:, 0]) * on
        if grad != "none":
            d = logp.exp_().sub_(target).mul_((s["g"][r:r + block].double() * on / temp)[:, None])
            dX[r:r + block] = torch.matmul(d, W)
            if dW is not None:
                dW.addmm_(d.T, x)
    out = {"loss": loss, "lse": lse}
    if grad != "none":
        out["dx"] = dX
        if grad == "both":
            out["dw"] = dW
    return out
