"""What is read off a row of logits beside its loss, and what a student learns from it: the cases
that these training operators are timed on.

A case is a dict of plain values.  Its "op" names the operator, its "dir" the direction:

    logprob  fwd   log probabilities of given tokens, each row's entropy and its top classes
             grad  the same, then the logits' gradient from theirs through autograd
    distill  fwd   each row's divergence from a teacher's top classes
             step  their mean and the gradient of the logits in one call
             grad  their mean, then the gradient through autograd

`run` computes them in their plain form where `own` is false, and through
defmuon_amd.train_ops where it is true.

With x = z / tau, lse = log sum exp x and p = exp(x - lse):

    log p_y = x_y - lse,    H = -sum p log p,    top: the largest log p, ties by the lower class

and for a teacher's list of classes i_j with log probabilities t_j,

    q = softmax(t),         loss = tau^2 sum_j q_j (log q_j - log p_{i_j})

or, with the rest of the classes as one more,

    q = exp(t), r = 1 - sum q,   loss = tau^2 (sum_j q_j (log q_j - log p_{i_j})
                                               + r (log r - log of p's sum over the rest))
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100


# ---- cases ----------------------------------------------------------------------------------

def _logprob(dir, rows, vocab, stride, dtype, top=0, tau=1.0, tokens=True, ignored=0.0):
    """stride: elements from row to row (classes padded for the product); ignored: share of rows
    whose token is not to be scored."""
    return {"op": "logprob", "dir": dir, "rows": rows, "vocab": vocab, "stride": stride,
            "dtype": dtype, "top": top, "tau": tau, "tokens": tokens, "ignored": ignored}


def _distill(dir, rows, vocab, stride, dtype, top, teacher="fp32", tau=1.0, rest=False,
             ignored=0.0, ragged=False):
    """top: length of the teacher's lists, and teacher their type; ragged: some end earlier."""
    return {"op": "distill", "dir": dir, "rows": rows, "vocab": vocab, "stride": stride,
            "dtype": dtype, "top": top, "teacher": teacher, "tau": tau, "rest": rest,
            "ignored": ignored, "ragged": ragged}


def listed():
    return [
        # the next token's alternatives while a model answers: launches and latency
        {"name": "logprob 1x50257 top 5", **_logprob("fwd", 1, 50257, 50304, "bf16", top=5)},
        # scoring an answer of a few hundred tokens, fp16 rows of odd length
        {"name": "logprob 341x32003", **_logprob("fwd", 341, 32003, 32003, "fp16", ignored=0.1)},
        # a teacher's pass over the 8 x 1024 tokens of a GPT-2 step, its top classes to keep
        {"name": "logprob 8192x50257 top 64",
         **_logprob("fwd", 8192, 50257, 50304, "bf16", top=64, tau=2.0, tokens=False)},
        # a larger vocabulary in fp32, with the alternatives that an evaluation reports
        {"name": "logprob 1000x131072 top 20",
         **_logprob("fwd", 1000, 131072, 131072, "fp32", top=20)},
        # learning from rewards: log probabilities and entropy with their gradient
        {"name": "logprob grad 4096x50257", **_logprob("grad", 4096, 50257, 50257, "bf16")},
        # ... a small model's in fp32, the alternatives' log probabilities among the outputs
        {"name": "logprob grad 333x8009 top 8",
         **_logprob("grad", 333, 8009, 8009, "fp32", top=8, tau=0.7, ignored=0.1)},
        # how far a student is from its teacher on a held-out text
        {"name": "distill 1024x50257", **_distill("fwd", 1024, 50257, 50304, "bf16", 32, rest=True)},
        # a student's step on a handful of answers
        {"name": "distill step 16x50257", **_distill("step", 16, 50257, 50304, "bf16", 16)},
        # GPT-2's training step on a teacher's lists, the rest of the classes as one
        {"name": "distill step 8192x50257",
         **_distill("step", 8192, 50257, 50257, "bf16", 64, tau=2.0, rest=True)},
        # a larger vocabulary, longer lists in half precision
        {"name": "distill step 2048x131072",
         **_distill("step", 2048, 131072, 131072, "bf16", 128, teacher="fp16")},
        # fp32 logits of a middling vocabulary, lists of different lengths, through autograd
        {"name": "distill grad 2000x32003",
         **_distill("grad", 2000, 32003, 32003, "fp32", 20, tau=1.5, rest=True, ignored=0.1,
                    ragged=True)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, dir = rng.choice([("logprob", "fwd"), ("logprob", "fwd"), ("logprob", "grad"),
                          ("distill", "fwd"), ("distill", "step"), ("distill", "grad")])
    vocab = _log_int(rng, 256, 131072)
    stride = vocab + (-vocab % 64 if rng.random() < 0.5 else 0)
    dtype = rng.choice(list(DTYPES))
    rows = _log_int(rng, 1, min(16384, 8192 * 50257 // (vocab * BYTES[dtype] // 2)))
    tau, ignored = rng.choice([1.0, 1.0, 0.7, 2.0]), rng.choice([0.0, 0.1])
    if op == "logprob":
        top = rng.choice([0, _log_int(rng, 1, 128)])
        tokens = top == 0 or rng.random() < 0.7
        return _logprob(dir, rows, vocab, stride, dtype, top, tau, tokens,
                        ignored if tokens else 0.0)
    return _distill(dir, rows, vocab, stride, dtype, _log_int(rng, 1, 128),
                    rng.choice(list(DTYPES)), tau, rng.random() < 0.5, ignored,
                    rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------------------------

def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    n, v, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=DEV)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    buf = torch.empty((n, case["stride"]), device=DEV, dtype=dt)
    for r in range(0, n, 1024):
        m = min(1024, n - r)
        buf[r:r + m] = normal(m, case["stride"]).mul_(2.0).to(dt)
    s = {"logits": buf[:, :v]}

    def lift(at, by):
        s["logits"].scatter_(1, at, (s["logits"].gather(1, at).float() + by).to(dt))

    # tokens whose frequencies fall as one over their rank, in a shuffled order of ranks
    rank = torch.exp(uniform(n).double() * math.log(v + 1.0)) - 1.0
    tokens = torch.randperm(v, generator=gen, device=DEV)[rank.long().clamp_(0, v - 1)]
    gone = uniform(n) < case["ignored"]
    gone[0] = False   # a mean has a row
    if case["op"] == "logprob":
        lift(tokens[:, None], uniform(n, 1) * 8.0)   # most rows know something of their token
        s["tokens"] = torch.where(gone, IGNORE, tokens) if case["tokens"] else None
        if case["dir"] == "grad":
            s["grads"] = (normal(n) / n if case["tokens"] else None, normal(n) * (0.01 / n),
                          normal(n, case["top"]) / n if case["top"] else None)
        return s
    k = min(case["top"], v)
    # distinct classes a row: a walk through all of them by a step that shares no factor with
    # their number
    steps = [t for t in range(1, min(v, 4096)) if math.gcd(t, v) == 1] or [1]
    step = torch.tensor(steps, device=DEV)[(uniform(n).double() * len(steps)).long()]
    ids = (tokens[:, None] + step[:, None] * torch.arange(k, device=DEV)) % v
    # the lists hold most of the teacher's mass, their values falling
    t = torch.sort(normal(n, k) * 2.0, dim=1, descending=True)[0]
    t = t - torch.logsumexp(t, 1, keepdim=True)
    lift(ids, t + 8.0 + normal(n, k))   # the student has learned some of it
    t = t + torch.log(0.6 + 0.399 * uniform(n, 1))
    if case["ragged"]:
        length = 1 + (uniform(n, 1) * 2.0 * k).long()
        ids = torch.where(torch.arange(k, device=DEV) < length, ids, IGNORE)
    s["ids"] = torch.where(gone[:, None], IGNORE, ids)
    s["teacher"] = t.to(DTYPES[case["teacher"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return s


# ---- one pass -------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _RUN_OWN[case["op"]](case, state)
    return _RUN_PLAIN[case["op"]](case, state)


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "spectral-deflation_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from defmuon_amd import train_ops
    return train_ops


def _given(outputs):
    return tuple(o for o in outputs if o is not None)


def _own_logprob(case, s):
    ops = _ops()
    kw = {"top": case["top"], "temperature": case["tau"], "ignore_index": IGNORE}
    if case["dir"] == "fwd":
        return _given(ops.token_log_probs(s["logits"], s["tokens"], **kw))
    z = s["logits"].detach().requires_grad_()
    out = ops.token_log_probs(z, s["tokens"], **kw)
    pairs = [(o, g) for o, g in zip(out, s["grads"]) if o is not None]
    dz = torch.autograd.grad([o for o, _ in pairs], z, [g for _, g in pairs])[0]
    return (*(o.detach() for o in _given(out)), dz)


def _own_distill(case, s):
    ops = _ops()
    kw = {"temperature": case["tau"], "rest": case["rest"], "ignore_index": IGNORE}
    if case["dir"] == "fwd":
        return ops.distillation(s["logits"], s["ids"], s["teacher"], reduction="none", **kw)
    if case["dir"] == "step":
        return ops.distillation_step(s["logits"], s["ids"], s["teacher"], **kw)
    z = s["logits"].detach().requires_grad_()
    loss = ops.distillation(z, s["ids"], s["teacher"], **kw)
    return loss.detach(), torch.autograd.grad(loss, z)[0]


_RUN_OWN = {"logprob": _own_logprob, "distill": _own_distill}


def _top(z, k):
    """The classes of the k largest of each row's fp32 logits, ties by the lower class: the
    largest of whole numbers that order first by value, then by class."""
    v, out = z.shape[1], []
    for zz in z.split(1024):
        bits = (zz + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = order * v + torch.arange(v - 1, -1, -1, device=DEV)
        out.append(v - 1 - torch.remainder(torch.topk(key, k, dim=1)[0], v))
    return torch.cat(out)


def _plain_logprob(case, s):
    z, tau, y, k = s["logits"].float(), case["tau"], s["tokens"], case["top"]
    zero = torch.zeros((), device=DEV)
    m = z.amax(1, keepdim=True)
    d = (z - m) / tau
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_s = torch.log(total)
    entropy = (log_s - (e * d).sum(1, keepdim=True) / total)[:, 0]
    out, live = [], None
    if y is not None:
        live = y != IGNORE
        at = torch.where(live, y, torch.zeros_like(y))[:, None]
        out.append(torch.where(live, (d.gather(1, at) - log_s)[:, 0], zero))
        entropy = torch.where(live, entropy, zero)
    out.append(entropy)
    ids = None
    if k:
        ids = _top(z, k)
        top = d.gather(1, ids) - log_s
        if live is not None:
            top = torch.where(live[:, None], top, zero)
        out += [top, ids if live is None else torch.where(live[:, None], ids, IGNORE)]
    if case["dir"] == "fwd":
        return tuple(out)
    gy, gh, gt = s["grads"]
    push = torch.zeros_like(total)
    if gy is not None:
        push = push + gy[:, None]
    if gt is not None:
        push = push + gt.sum(1, keepdim=True)
    p = e / total
    dz = -p * (push + gh[:, None] * ((d - log_s) + entropy[:, None]))
    if gy is not None:
        dz.scatter_add_(1, at, gy[:, None])
    if gt is not None:
        dz.scatter_add_(1, ids, gt)
    if live is not None:
        dz = torch.where(live[:, None], dz, zero)
    return (*out, (dz / tau).to(s["logits"].dtype))


def _plain_distill(case, s):
    tau, ids, v = case["tau"], s["ids"], case["vocab"]
    x = s["logits"].float() / tau
    zero = torch.zeros((), device=DEV)
    some = ids != IGNORE
    live = some[:, :1]
    t = torch.where(some, s["teacher"].float(), -torch.inf)
    at = torch.where(some, ids, torch.zeros_like(ids))
    q = torch.exp(t) if case["rest"] else torch.softmax(torch.where(live, t, zero), 1)
    log_p = x - torch.logsumexp(x, 1, keepdim=True)
    part = torch.where(q > 0, q * (torch.log(q) - log_p.gather(1, at)), zero)
    loss = part.sum(1, keepdim=True)
    share = q.sum(1, keepdim=True)
    if case["rest"]:
        in_list = torch.zeros((x.shape[0], v + 1), device=DEV, dtype=torch.bool)
        in_list.scatter_(1, torch.where(some, ids, v), True)
        others = torch.where(in_list[:, :v], -torch.inf, x)
        log_o = torch.logsumexp(others, 1, keepdim=True)
        left = torch.clamp(1.0 - share, min=0.0)
        gap = torch.log(left) - (log_o - torch.logsumexp(x, 1, keepdim=True))
        loss = loss + torch.where(left > 0, left * gap, zero)
        share = share + left
    loss = torch.where(live, loss * tau ** 2, zero)[:, 0]
    if case["dir"] == "fwd":
        return loss
    count = live.sum()
    dz = torch.exp(log_p) * share
    dz.scatter_add_(1, at, torch.where(some, -q, zero))
    if case["rest"]:
        dz -= left * torch.exp(others - log_o)
    dz = torch.where(live, dz * tau, zero) / count
    return loss.sum() / count, dz.to(s["logits"].dtype)


_RUN_PLAIN = {"logprob": _plain_logprob, "distill": _plain_distill}


# ---- the least a pass moves and computes ----------------------------------------------------

def work(case):
    n, numel = case["rows"], case["rows"] * case["vocab"]
    passes = 1 if case["dir"] == "fwd" else 2
    bytes_, flops = numel * BYTES[case["dtype"]] * passes, 6 * numel * passes
    if case["op"] == "logprob":
        bytes_ += n * (4 + 12 * case["tokens"] + 12 * case["top"])
        if case["dir"] == "grad":
            bytes_ += n * 4 * (1 + case["tokens"] + case["top"])
    else:
        bytes_ += n * (4 + case["top"] * (8 + BYTES[case["teacher"]]))
    return {"bytes": bytes_, "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------------------

def exact(case, seed):
    """Row by row in float64, gradients by differentiating the definitions."""
    s = _inputs(case, seed)
    parts = []
    wanted = case["dir"] != "fwd"
    for r in range(0, case["rows"], 256):
        rows = slice(r, min(r + 256, case["rows"]))
        z = s["logits"][rows].double().requires_grad_(wanted)
        parts.append((_exact_logprob if case["op"] == "logprob" else _exact_distill)
                     (case, s, rows, z))
    whole = [torch.cat([p[i] for p in parts]) for i in range(len(parts[0]))]
    if case["op"] == "logprob":
        return tuple(whole)
    if not wanted:
        return whole[0]
    count = int((s["ids"][:, 0] != IGNORE).sum())
    return whole[0].sum() / count, whole[1] / count


def _exact_logprob(case, s, rows, z):
    x = torch.log_softmax(z / case["tau"], dim=1)
    y = None if s["tokens"] is None else s["tokens"][rows]
    n = z.shape[0]
    keep = torch.ones(n, device=DEV, dtype=torch.bool) if y is None else y != IGNORE
    mask = keep.double()
    outs = []
    if y is not None:
        outs.append(x[torch.arange(n, device=DEV), y * keep] * mask)
    outs.append(torch.special.entr(torch.softmax(z / case["tau"], dim=1)).sum(1) * mask)
    ids = None
    if case["top"]:
        ids = torch.sort(s["logits"][rows].float(), dim=1, descending=True,
                         stable=True)[1][:, :case["top"]]
        outs.append(x.gather(1, ids) * mask[:, None])
    result = [o.detach() for o in outs]
    if ids is not None:
        result.append(torch.where(keep[:, None], ids, IGNORE))
    if case["dir"] == "grad":
        given = [g[rows].double() for g in s["grads"] if g is not None]
        result.append(torch.autograd.grad(outs, z, given)[0])
    return result


def _exact_distill(case, s, rows, z):
    v = case["vocab"]
    ids, t = s["ids"][rows], s["teacher"][rows].double()
    some = ids != IGNORE
    t = t.masked_fill(~some, -torch.inf)
    live = some[:, 0]
    # the teacher's distribution over all classes, a column more for what is left out
    q = torch.exp(t) if case["rest"] else torch.exp(t - torch.logsumexp(t, 1, keepdim=True))
    q = torch.nan_to_num(q)
    wide = torch.zeros((z.shape[0], v + 1), device=DEV, dtype=torch.float64)
    wide.scatter_(1, ids.masked_fill(~some, v), q)
    listed_ = torch.zeros_like(wide)
    listed_.scatter_(1, ids.masked_fill(~some, v), 1.0)
    x = torch.log_softmax(z / case["tau"], dim=1)
    dense = wide[:, :v]
    loss = torch.special.xlogy(dense, dense).sum(1) - (dense * x).sum(1)
    if case["rest"]:
        left = (1.0 - dense.sum(1)).clamp(min=0.0)
        others = torch.logsumexp(x.masked_fill(listed_[:, :v] > 0, -torch.inf), 1)
        loss = loss + torch.special.xlogy(left, left) - left * others
    loss = loss * live.double() * case["tau"] ** 2
    if case["dir"] == "fwd":
        return [loss.detach()]
    return [loss.detach(), torch.autograd.grad(loss.sum(), z)[0]]
