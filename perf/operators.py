"""The training operators beside the optimizer, and what they are timed on.

A case is a dict of plain values.  Its "op" names the operator, its "dir" the direction:

    embed    fwd   token rows times a scale, plus position rows, through dropout
             bwd   the gradients of both tables from the gradient of the output
    dropout  fwd   dropout by a counter-based generator, plus a residual
             bwd   the gradient of its input, with the same mask
    xent     fwd   cross entropy of each row over the classes
             step  mean loss and the gradient of the logits in one call
             grad  mean loss, then the gradient through autograd

`run` computes them in their plain form where `own` is false, and through
defmuon_amd.train_ops where it is true.

Dropout: element e of a tensor (flat index) takes half (e & 1) of word (e >> 1) & 3 of the
Philox4x32-10 block (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
1, 2, 3", SC 2011) with counter (e >> 3, offset) and key seed, low words first.  It is kept
if these 16 bits are at least t = round(65536 p), and then scaled by 65536 / (65536 - t).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100


# ---- cases ----------------------------------------------------------------------------------

def _embed(dir, batch, seq, dim, vocab, ctx, dtype, out, scale=1.0, p=0.0, pad=False):
    """dtype: of the tables (fwd) or of the incoming gradient (bwd); out: of the outputs;
    ctx: rows of the position table, 0 for none; pad: token 0 is padding."""
    return {"op": "embed", "dir": dir, "batch": batch, "seq": seq, "dim": dim, "vocab": vocab,
            "ctx": ctx, "dtype": dtype, "out": out, "scale": scale, "p": p, "pad": pad}


def _dropout(dir, rows, dim, dtype, residual="", p=0.1):
    """residual: its type, which is the output's too; empty for none."""
    return {"op": "dropout", "dir": dir, "rows": rows, "dim": dim, "dtype": dtype,
            "residual": residual, "p": p}


def _xent(dir, rows, vocab, stride, dtype, ignored=0.0, smooth=0.0, z=0.0):
    """stride: elements from row to row (classes padded for the product); ignored: share of
    rows without a target."""
    return {"op": "xent", "dir": dir, "rows": rows, "vocab": vocab, "stride": stride,
            "dtype": dtype, "ignored": ignored, "smooth": smooth, "z": z}


def listed():
    return [
        # a prompt's first token through a model kept in bf16: launches and latency
        {"name": "embed one token", **_embed("fwd", 1, 1, 768, 50257, 1024, "bf16", "bf16")},
        # the input of a GPT-2-large training step: fp32 tables, embedding dropout
        {"name": "embed 8x1024x1280",
         **_embed("fwd", 8, 1024, 1280, 50257, 1024, "fp32", "fp32", p=0.1)},
        # a ragged batch of a small model with scaled fp16 tables and no positions
        {"name": "embed ragged 3x341x771",
         **_embed("fwd", 3, 341, 771, 8009, 0, "fp16", "fp16", scale=math.sqrt(771))},
        # a short padded batch of a toy model: the gradient's launches
        {"name": "embed grad 2x77x192",
         **_embed("bwd", 2, 77, 192, 1009, 128, "fp32", "fp32", pad=True)},
        # the gradient of GPT-2 large's embedding in one step of 8 x 1024 tokens
        {"name": "embed grad 8x1024x1280",
         **_embed("bwd", 8, 1024, 1280, 50257, 1024, "fp32", "fp32", p=0.1)},
        # ... and of the 32 x 1024 tokens that one GPU takes of a large batch, bf16 stream
        {"name": "embed grad 32x1024x1280",
         **_embed("bwd", 32, 1024, 1280, 50257, 1024, "bf16", "fp32")},
        # a short sequence's residual addition: latency
        {"name": "dropout 64x768", **_dropout("fwd", 64, 768, "bf16", "bf16")},
        # the residual addition of a GPT-2-large block under autocast
        {"name": "dropout 8192x1280", **_dropout("fwd", 8192, 1280, "bf16", "fp32")},
        # the gradient of dropout on an MLP's hidden values
        {"name": "dropout grad 8192x5120", **_dropout("bwd", 8192, 5120, "bf16", p=0.2)},
        # losses of a handful of answers, classes padded to a multiple of 64
        {"name": "xent 16x50257", **_xent("fwd", 16, 50257, 50304, "bf16")},
        # the loss of a GPT-2-large training step and its gradient
        {"name": "xent step 8192x50257", **_xent("step", 8192, 50257, 50257, "bf16")},
        # fp32 logits of a middling vocabulary, every option, through autograd
        {"name": "xent grad 2000x32003",
         **_xent("grad", 2000, 32003, 32003, "fp32", ignored=0.1, smooth=0.1, z=1e-4)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, dir = rng.choice([("embed", "fwd"), ("embed", "bwd"), ("dropout", "fwd"),
                          ("dropout", "bwd"), ("xent", "fwd"), ("xent", "step"),
                          ("xent", "grad")])
    if op == "embed":
        dim = _log_int(rng, 64, 1600)
        if rng.random() < 0.5:
            dim -= dim % 64
        tokens = _log_int(rng, 1, 32768 * 1280 // max(dim, 1280))
        seq = min(tokens, _log_int(rng, 1, 1024))
        vocab = _log_int(rng, 256, min(131072, 50257 * 1280 // dim))
        dtype, out = rng.choice([("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"),
                                 ("fp32", "bf16"), ("bf16", "fp32")])
        return _embed(dir, tokens // seq, seq, dim, vocab,
                      rng.choice([0, seq, 1024]), dtype, out,
                      scale=rng.choice([1.0, math.sqrt(dim)]), p=rng.choice([0.0, 0.1, 0.25]),
                      pad=rng.random() < 0.25)
    if op == "dropout":
        dim = _log_int(rng, 64, 5120)
        if rng.random() < 0.5:
            dim -= dim % 64
        rows = _log_int(rng, 1, min(32768, 8192 * 5120 // dim))
        dtype = rng.choice(list(DTYPES))
        residual = rng.choice(["", dtype, "fp32"]) if dir == "fwd" else ""
        return _dropout(dir, rows, dim, dtype, residual, p=rng.choice([0.05, 0.1, 0.2, 0.5]))
    vocab = _log_int(rng, 256, 131072)
    stride = vocab + (-vocab % 64 if rng.random() < 0.5 else 0)
    dtype = rng.choice(list(DTYPES))
    rows = _log_int(rng, 1, min(16384, 8192 * 50257 // (vocab * BYTES[dtype] // 2)))
    return _xent(dir, rows, vocab, stride, dtype, ignored=rng.choice([0.0, 0.1]),
                 smooth=rng.choice([0.0, 0.1]), z=rng.choice([0.0, 1e-4]))


# ---- inputs ---------------------------------------------------------------------------------

def _tokens(gen, shape, vocab):
    """Ids whose frequencies fall as one over their rank, in a shuffled order of ranks."""
    u = torch.rand(shape, generator=gen, device=DEV, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=gen, device=DEV)[rank]


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(std).to(dtype)

    s = {"rng": (int(seed) * 0x9E3779B97F4A7C15 % (1 << 63), 5)}
    if case["op"] == "embed":
        shape = (case["batch"], case["seq"])
        s["ids"] = _tokens(gen, shape, case["vocab"])
        if case["pad"]:   # every sequence ends in a few padding tokens
            s["ids"][:, case["seq"] - case["seq"] // 8:] = 0
        if case["dir"] == "fwd":
            s["weight"] = normal(case["vocab"], case["dim"], std=0.02)
            s["pos"] = normal(case["ctx"], case["dim"], std=0.01) if case["ctx"] else None
        else:
            s["grad"] = normal(*shape, case["dim"], std=1e-2)
    elif case["op"] == "dropout":
        s["x"] = normal(case["rows"], case["dim"])
        if case["residual"]:
            s["residual"] = normal(case["rows"], case["dim"], dtype=DTYPES[case["residual"]])
    else:
        n, v = case["rows"], case["vocab"]
        s["targets"] = _tokens(gen, (n,), v)
        buf = torch.empty((n, case["stride"]), device=DEV, dtype=dt)
        for r in range(0, n, 1024):
            m = min(1024, n - r)
            buf[r:r + m] = normal(m, case["stride"], std=2.0)
        s["logits"] = buf[:, :v]
        # most rows know something of their target
        bonus = torch.rand((n, 1), generator=gen, device=DEV) * 8.0
        at = s["targets"][:, None]
        s["logits"].scatter_(1, at, (s["logits"].gather(1, at).float() + bonus).to(dt))
        if case["ignored"]:
            gone = torch.rand((n,), generator=gen, device=DEV) < case["ignored"]
            gone[0] = False   # the mean has a row
            s["targets"][gone] = IGNORE
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


def _own_embed(case, s):
    ops = _ops()
    kw = {"scale": case["scale"], "padding_idx": 0 if case["pad"] else None,
          "dropout_p": case["p"], "rng": s["rng"]}
    if case["dir"] == "fwd":
        return ops.embedding(s["ids"], s["weight"], s["pos"], out_dtype=DTYPES[case["out"]], **kw)
    dw, dp = ops.embedding_backward(s["grad"], s["ids"], case["vocab"], pos_rows=case["ctx"],
                                    dtype=DTYPES[case["out"]], **kw)
    return (dw,) if dp is None else (dw, dp)


def _own_dropout(case, s):
    ops = _ops()
    if case["dir"] == "fwd":
        return ops.dropout(s["x"], case["p"], s["rng"], residual=s.get("residual"))
    return ops.dropout_backward(s["x"], case["p"], s["rng"])


def _own_xent(case, s):
    ops = _ops()
    kw = {"ignore_index": IGNORE, "label_smoothing": case["smooth"], "z_loss": case["z"]}
    if case["dir"] == "fwd":
        return ops.cross_entropy(s["logits"], s["targets"], reduction="none", **kw)
    if case["dir"] == "step":
        return ops.cross_entropy_step(s["logits"], s["targets"], **kw)
    z = s["logits"].detach().requires_grad_()
    loss = ops.cross_entropy(z, s["targets"], reduction="mean", **kw)
    return loss.detach(), torch.autograd.grad(loss, z)[0]


_RUN_OWN = {"embed": _own_embed, "dropout": _own_dropout, "xent": _own_xent}


def _keep(shape, p, rng):
    """Truth values of the kept elements, and the scale of what is kept."""
    numel = math.prod(shape)
    low = 0xFFFFFFFF
    n = torch.arange((numel + 7) // 8, device=DEV, dtype=torch.int64)
    c = [n & low, n >> 32, torch.full_like(n, rng[1] & low), torch.full_like(n, rng[1] >> 32)]
    k0, k1 = rng[0] & low, rng[0] >> 32
    for _ in range(10):
        # 32 x 32 -> 64 bits: int64 products wrap, their bits are those of uint64
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    draws = torch.stack([half for w in c for half in (w & 0xFFFF, w >> 16)], dim=1)
    t = int(round(p * 65536))
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return (draws >= t).reshape(-1)[:numel].reshape(shape), scale


def _drop(x, p, rng):
    """Dropout of an fp32 tensor, itself where p is 0."""
    if p == 0:
        return x
    keep, scale = _keep(x.shape, p, rng)
    return torch.where(keep, x * scale, torch.zeros((), device=DEV))


def _plain_embed(case, s):
    dt = DTYPES[case["out"]]
    if case["dir"] == "fwd":
        x = s["weight"][s["ids"]].float() * case["scale"]
        if s["pos"] is not None:
            x = x + s["pos"][:case["seq"]].float()
        return _drop(x, case["p"], s["rng"]).to(dt)
    g = _drop(s["grad"].float(), case["p"], s["rng"])
    rows, ids = g.reshape(-1, case["dim"]) * case["scale"], s["ids"].reshape(-1)
    if case["pad"]:
        rows = torch.where(ids[:, None] == 0, torch.zeros((), device=DEV), rows)
    dw = torch.zeros((case["vocab"], case["dim"]), device=DEV).index_add_(0, ids, rows)
    if not case["ctx"]:
        return (dw.to(dt),)
    dp = torch.zeros((case["ctx"], case["dim"]), device=DEV)
    dp[:case["seq"]] = g.sum(0)
    return dw.to(dt), dp.to(dt)


def _plain_dropout(case, s):
    y = _drop(s["x"].float(), case["p"], s["rng"])
    if case["dir"] == "fwd" and case["residual"]:
        return (y + s["residual"].float()).to(s["residual"].dtype)
    return y.to(s["x"].dtype)


def _plain_xent(case, s):
    z, y, v, eps = s["logits"].float(), s["targets"], case["vocab"], case["smooth"]
    valid = y != IGNORE
    at = torch.where(valid, y, torch.zeros_like(y))[:, None]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    loss = (lse - (1 - eps) * z.gather(1, at) - eps * z.mean(1, keepdim=True)
            + case["z"] * lse * lse)[:, 0]
    loss = torch.where(valid, loss, torch.zeros_like(loss))
    if case["dir"] == "fwd":
        return loss
    count = valid.sum()
    dz = e * ((1 + 2 * case["z"] * lse) / total) - eps / v
    dz.scatter_add_(1, at, torch.full_like(lse, eps - 1))
    dz = torch.where(valid[:, None], dz / count, torch.zeros((), device=DEV))
    return loss.sum() / count, dz.to(s["logits"].dtype)


_RUN_PLAIN = {"embed": _plain_embed, "dropout": _plain_dropout, "xent": _plain_xent}


# ---- the least a pass moves and computes ----------------------------------------------------

def _distinct(tokens, vocab):
    """Expected count of different ids among `tokens` of _tokens."""
    edge = np.log(np.arange(1, vocab + 2, dtype=np.float64)) / math.log(vocab + 1.0)
    return float(np.sum(1.0 - (1.0 - np.diff(edge)) ** tokens))


def work(case):
    if case["op"] == "embed":
        tokens, dim = case["batch"] * case["seq"], case["dim"]
        b, o = BYTES[case["dtype"]], BYTES[case["out"]]
        if case["dir"] == "fwd":
            rows = _distinct(tokens, case["vocab"]) + (case["seq"] if case["ctx"] else 0)
            return {"bytes": 8 * tokens + rows * dim * b + tokens * dim * o,
                    "flops": 3 * tokens * dim}
        return {"bytes": 8 * tokens + tokens * dim * b + (case["vocab"] + case["ctx"]) * dim * o,
                "flops": 3 * tokens * dim}
    if case["op"] == "dropout":
        b = BYTES[case["dtype"]]
        moved = 2 * b if not case["residual"] else b + 2 * BYTES[case["residual"]]
        return {"bytes": case["rows"] * case["dim"] * moved, "flops": 2 * case["rows"] * case["dim"]}
    numel = case["rows"] * case["vocab"]
    passes = 1 if case["dir"] == "fwd" else 2
    return {"bytes": numel * BYTES[case["dtype"]] * passes + 12 * case["rows"],
            "flops": 4 * numel * passes}


# ---- the definition in 64 bits --------------------------------------------------------------

def _exact_scale(shape, p, rng):
    """What dropout multiplies each element by, in float64, block by block in numpy."""
    size = int(np.prod(shape))
    blocks = np.arange(-(-size // 8), dtype=np.uint64)
    mask, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    x0, x1 = blocks & mask, blocks >> sh
    x2 = np.full_like(blocks, rng[1] % 2**32)
    x3 = np.full_like(blocks, rng[1] // 2**32)
    key = [rng[0] % 2**32, rng[0] // 2**32]
    for _ in range(10):
        left, right = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = ((right >> sh) ^ x1 ^ np.uint64(key[0]), right & mask,
                          (left >> sh) ^ x3 ^ np.uint64(key[1]), left & mask)
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    words = np.stack([x0, x1, x2, x3], axis=1).astype("<u4")
    draws = words.view("<u2").reshape(-1)[:size].reshape(shape)
    cut = int(round(p * 65536))
    keep = torch.from_numpy(draws.astype(np.int32)).to(DEV) >= cut
    return keep.double() * (65536.0 / (65536 - cut))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "embed":
        shape = (case["batch"], case["seq"], case["dim"])
        factor = _exact_scale(shape, case["p"], s["rng"]) if case["p"] else 1.0
        if case["dir"] == "fwd":
            x = case["scale"] * torch.index_select(s["weight"], 0, s["ids"].flatten()).double()
            x = x.view(shape)
            if case["ctx"]:
                x += s["pos"].double()[None, :case["seq"]]
            return x * factor
        g = s["grad"].double() * factor
        # sums of each id's rows as differences of one running sum over the sorted tokens
        ids, order = torch.sort(s["ids"].flatten())
        running = torch.cumsum(g.view(-1, case["dim"])[order], 0)
        running = torch.cat([torch.zeros_like(running[:1]), running])
        v = torch.arange(case["vocab"], device=DEV)
        dw = running[torch.searchsorted(ids, v, right=True)] - running[torch.searchsorted(ids, v)]
        dw *= case["scale"]
        if case["pad"]:
            dw[0] = 0
        if not case["ctx"]:
            return (dw,)
        dp = torch.zeros((case["ctx"], case["dim"]), device=DEV, dtype=torch.float64)
        for b in range(case["batch"]):
            dp[:case["seq"]] += g[b]
        return dw, dp
    if case["op"] == "dropout":
        y = s["x"].double() * _exact_scale(s["x"].shape, case["p"], s["rng"])
        return y + s["residual"].double() if case["residual"] else y
    y, v, eps, zeta = s["targets"], case["vocab"], case["smooth"], case["z"]
    count = int((y != IGNORE).sum())
    losses = torch.zeros(case["rows"], device=DEV, dtype=torch.float64)
    dz = None
    if case["dir"] != "fwd":
        dz = torch.zeros((case["rows"], v), device=DEV, dtype=torch.float64)
    want = torch.arange(v, device=DEV)
    for r in range(0, case["rows"], 512):
        z, t = s["logits"][r:r + 512].double(), y[r:r + 512]
        live = (t != IGNORE).double()
        q = (1 - eps) * (want[None, :] == t[:, None]).double() + eps / v
        lse = torch.logsumexp(z, 1)
        losses[r:r + 512] = live * (lse - (q * z).sum(1) + zeta * lse ** 2)
        if dz is not None:
            p = torch.exp(z - lse[:, None])
            dz[r:r + 512] = (p * (1 + 2 * zeta * lse[:, None]) - q) * live[:, None] / count
    return losses if dz is None else (losses.sum() / count, dz)
