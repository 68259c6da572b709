"""The operators of a GPT-2 training step beside its matrix products and the optimizer: the
embedding with its gradient, dropout, and the loss with its gradient; and beside the loss, on the
same rows of logits, log probabilities with entropy and top classes, and distillation from a
teacher's, with their gradients.

    x = embedding(tokens, wte, wpe, dropout_p=0.1, rng=draw_rng())
    x = dropout(attn(x), 0.1, draw_rng(), residual=x)
    loss, dlogits = cross_entropy_step(logits, targets)
    logits.backward(dlogits)

    top = token_log_probs(teacher(tokens), top=64, temperature=2.0)
    loss, dlogits = distillation_step(logits, top.top_ids, top.top_log_probs, temperature=2.0)

fp32, bf16 and fp16 tensors; everything is computed in fp32 and rounded once.  All functions
run through the HIP library on the current stream and synchronise nothing; there is no CPU
fallback.  embedding, dropout, cross_entropy, token_log_probs and distillation take part in
autograd; the *_backward and *_step functions are for programs that call the gradients themselves.
Arguments that do not fit raise NativeError, as do tensors that carry a forward-mode tangent:
there is no such derivative.  So do traces that would record the results' allocation and not the
launch behind it: make_fx and fake tensors for all functions, torch.jit.trace (which records
autograd functions) for those outside autograd.

Random numbers: `rng` names the mask of a dropout.  It is a pair of integers (seed, offset), or
an int64 tensor of the two on the GPU, which is read when a kernel runs: a captured graph
draws a new mask at each replay if the program changes the tensor between its replays (after
the backward pass, which reads it again; a change before raises torch's error for saved tensors).
The rows of a (layers, 2) tensor serve a model:
different offsets, and the seeds set anew by one operation.  A pair of integers would be the
same at every replay, so draw_rng, and with it Dropout without an rng, raises NativeError while a
graph is captured.  Two calls with
the same pair, shape and p drop the same elements, which is how the backward pass has its mask
without storing it; calls that should differ take different pairs (draw_rng).  p is taken to
the nearest 1/65536, and kept elements are scaled by the reciprocal of exactly that.  A dropped
element is replaced by zero, also where it is not finite.
"""

import collections

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from defmuon_amd import _native
from defmuon_amd._native import FLOATS, NativeError

__all__ = ["embedding", "embedding_backward", "dropout", "dropout_backward", "Dropout",
           "draw_rng", "cross_entropy", "cross_entropy_step", "token_log_probs", "TokenLogProbs",
           "distillation", "distillation_step"]

_is_tracing = torch._C._is_tracing
_modes = torch._C._len_torch_dispatch_stack
# the tracing mode of make_fx(pre_dispatch=True) is the first of a list of torch's own
_early_modes = vars(torch._ops._mode_stack_state_for_pre_dispatch).get(
    "_ModeStackStateForPreDispatch__infra_modes", [None])

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_NO_RNG = (0, 0, 0)


# ---- arguments ------------------------------------------------------------------------------

def _no_tangent(t, what, name):
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NativeError(f"{what}: no forward-mode derivative ({name} has a tangent)")


def _eager(what, function=False):
    """Refuse to be traced (function: torch.jit.trace records an autograd function instead)."""
    if not function and _is_tracing():
        raise NativeError(f"{what}: torch.jit.trace cannot record a launch")
    traced = _early_modes[0] is not None
    if _modes():
        key, mode = torch._C._TorchDispatchModeKey, torch._C._get_dispatch_mode
        traced |= mode(key.PROXY) is not None or mode(key.FAKE) is not None
    if traced:
        raise NativeError(f"{what}: a trace of torch calls cannot record a launch")


def _float(t, what, name):
    if forward_ad._current_level >= 0:
        _no_tangent(t, what, name)
    if not t.is_cuda:
        raise NativeError(f"{what}: the HIP path needs a GPU tensor ({name} is on {t.device})")
    if t.dtype not in FLOATS:
        raise NativeError(f"{what}: {name} must be fp32, bf16 or fp16, not {t.dtype}")


def _ints(t, device, what, name):
    if t.device != device:
        raise NativeError(f"{what}: {name} is on {t.device}, not on {device}")
    if t.dtype not in (torch.int64, torch.int32):
        raise NativeError(f"{what}: {name} must be int64 or int32, not {t.dtype}")


def _out_type(dtype, what):
    if dtype not in FLOATS:
        raise NativeError(f"{what}: the result's type must be fp32, bf16 or fp16, not {dtype}")


def _rows(t):
    """(tensor, rows, columns, row stride) of a tensor taken as rows of its last dimension; a
    copy where its rows are not contiguous or not evenly spaced."""
    cols = int(t.shape[-1]) if t.ndim else 1   # (a trace's sizes are tensors)
    rows = int(t.numel()) // cols if cols else 0
    if t.is_contiguous():
        return t, rows, cols, cols
    if t.stride(-1) == 1 or cols == 1:
        stride = inner = None
        for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if stride is None:
                stride, inner = st, st * size
            elif st == inner:
                inner = st * size
            else:
                break
        else:
            return t, rows, cols, cols if stride is None else stride
    return t.contiguous(), rows, cols, cols


def _drop(p, rng, like, what):
    """(cut, (seed, offset, state address)) of a dropout on `like`'s device."""
    if not 0.0 <= p <= 1.0:
        raise NativeError(f"{what}: p must be between 0 and 1, not {p}")
    cut = int(round(p * 65536))
    if cut == 0:
        return 0, _NO_RNG
    if isinstance(rng, torch.Tensor):
        if (rng.device != like.device or rng.dtype != torch.int64 or rng.shape != (2,)
                or not rng.is_contiguous()):
            raise NativeError(f"{what}: rng must be two int64 on {like.device}")
        return cut, (0, 0, rng.data_ptr())
    try:
        seed, offset = rng
        return cut, (int(seed) & (1 << 64) - 1, int(offset) & (1 << 64) - 1, 0)
    except (TypeError, ValueError):
        raise NativeError(f"{what}: dropout needs rng=(seed, offset), got {rng!r}") from None


def draw_rng():
    """A fresh (seed, offset) from torch's CPU generator: torch.manual_seed fixes it, and
    activation checkpointing draws the same one again when it repeats a forward pass.  Not in a
    captured graph or a trace, which would repeat it."""
    if _is_tracing() or torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        raise NativeError("draw_rng: a captured graph or a trace would repeat one mask; give "
                          "dropout an rng tensor")
    return tuple(torch.randint(-1 << 63, (1 << 63) - 1, (2,), device="cpu").tolist())


# ---- dropout --------------------------------------------------------------------------------

def _dropout(x, residual, cut, rng, dtype):
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        like = x if dtype == x.dtype else residual
        out = torch.empty_like(like) if like is not None and like.dtype == dtype else (
            torch.empty_like(x, dtype=dtype))
        n = x.numel()
        if n:
            _native.dropout(x, residual, out, cut, rng, (1, n, n, n))
        return out
    out = torch.empty(x.shape, dtype=dtype, device=x.device)
    if out.numel():
        x, rows, cols, stride = _rows(x)
        rstride = 0
        if residual is not None:
            residual, _, _, rstride = _rows(residual)
        _native.dropout(x, residual, out, cut, rng, (rows, cols, stride, rstride))
    return out


class _Dropout(Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng):
        ctx.p, ctx.rng, ctx.dtype = p, rng, x.dtype
        if isinstance(rng, torch.Tensor):   # saved: autograd says so if it has changed
            ctx.save_for_backward(rng)
            ctx.rng = None
        cut, key = _drop(p, rng, x, "dropout")
        return _dropout(x, residual, cut, key, x.dtype if residual is None else residual.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        dx = None
        if ctx.needs_input_grad[0]:
            rng = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.rng
            dx = dropout_backward(grad, ctx.p, rng, ctx.dtype)
        return dx, grad if ctx.needs_input_grad[1] else None, None, None


def dropout(x, p, rng, residual=None):
    """Dropout of x, plus `residual` (same shape; the result then has its type)."""
    _eager("dropout", function=True)
    _float(x, "dropout", "x")
    if residual is not None:
        _float(residual, "dropout", "residual")
        if residual.shape != x.shape or residual.device != x.device:
            raise NativeError(f"dropout: residual is {tuple(residual.shape)} on "
                              f"{residual.device}, x {tuple(x.shape)} on {x.device}")
    cut, key = _drop(p, rng, x, "dropout")
    if _is_tracing() or torch.is_grad_enabled() and (
            x.requires_grad or residual is not None and residual.requires_grad):
        return _Dropout.apply(x, residual, p, rng)
    return _dropout(x, residual, cut, key, x.dtype if residual is None else residual.dtype)


def dropout_backward(grad, p, rng, dtype=None):
    """The gradient of dropout's x (in `dtype`, the gradient's own by default); that of its
    residual is `grad` itself."""
    _eager("dropout_backward")
    _float(grad, "dropout_backward", "grad")
    dtype = dtype or grad.dtype
    _out_type(dtype, "dropout_backward")
    return _dropout(grad, None, *_drop(p, rng, grad, "dropout_backward"), dtype)


class Dropout(torch.nn.Module):
    """Dropout and an optional residual's addition; in training a mask of its own at each call,
    or that of `rng` (which a captured graph needs, as a tensor), in evaluation x (+ residual)."""

    def __init__(self, p=0.1):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise NativeError(f"Dropout: p must be between 0 and 1, not {p}")
        self.p = p

    def extra_repr(self):
        return f"p={self.p}"

    def forward(self, x, residual=None, rng=None):
        p = self.p if self.training else 0.0
        if p == 0.0 and residual is None:
            return x
        return dropout(x, p, draw_rng() if p and rng is None else rng, residual)


# ---- embedding ------------------------------------------------------------------------------

def _table(t):
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _positions(positions, ids, what):
    """(ids, positions) as the kernels take them, both of the wider type of the two."""
    if positions is None:
        return ids, None
    _ints(positions, ids.device, what, "positions")
    if positions.shape != ids.shape:
        raise NativeError(f"{what}: positions are {tuple(positions.shape)}, ids "
                          f"{tuple(ids.shape)}")
    if positions.dtype != ids.dtype:
        ids, positions = ids.long(), positions.long()
    return ids, positions.contiguous()


def _embed(ids, weight, pos_weight, positions, scale, cut, key, dtype):
    shape = (*ids.shape, weight.shape[1])
    out = weight.new_empty(shape) if dtype == weight.dtype else torch.empty(
        shape, dtype=dtype, device=weight.device)
    if out.numel():
        _native.embedding(ids.contiguous(), _table(weight),
                          None if pos_weight is None else _table(pos_weight), positions, scale,
                          cut, key, out)
    return out


class _Embedding(Function):
    @staticmethod
    def forward(ctx, weight, pos_weight, ids, positions, scale, padding_idx, p, rng, dtype):
        tensor = isinstance(rng, torch.Tensor)   # saved: autograd says so if it has changed
        ctx.save_for_backward(ids, positions, rng if tensor else None)
        ctx.args = scale, padding_idx, p, None if tensor else rng
        ctx.weight = weight.shape[0], weight.dtype
        ctx.pos = None if pos_weight is None else (pos_weight.shape[0], pos_weight.dtype)
        cut, key = _drop(p, rng, weight, "embedding")
        return _embed(ids, weight, pos_weight, positions, scale, cut, key, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ids, positions, state = ctx.saved_tensors
        scale, padding_idx, p, rng = ctx.args
        need_w, need_p = ctx.needs_input_grad[:2]
        dw, dp = embedding_backward(
            grad, ids, ctx.weight[0] if need_w else 0, pos_rows=ctx.pos[0] if need_p else 0,
            positions=positions, scale=scale, padding_idx=padding_idx if need_w else None,
            dropout_p=p, rng=rng if state is None else state, dtype=ctx.weight[1])
        return dw if need_w else None, dp if need_p else None, *[None] * 7


def embedding(ids, weight, pos_weight=None, positions=None, scale=1.0, padding_idx=None,
              dropout_p=0.0, rng=None, out_dtype=None):
    """dropout(scale * weight[ids] + pos_weight[positions]): (*ids.shape, dim).

    ids: int64 or int32; positions: of ids' shape, by default the index along its last
    dimension.  The tables have one type; out_dtype is theirs by default.  padding_idx takes no
    gradient.  An id or position outside its table gives a row of NaN."""
    what = "embedding"
    _eager(what, function=True)
    _float(weight, what, "weight")
    device, dtype, shape = weight.device, weight.dtype, weight.shape
    if len(shape) != 2:
        raise NativeError(f"{what}: weight must be (rows, dim), got {tuple(shape)}")
    if shape[1] > 1 << 30 or pos_weight is not None and ids.ndim and ids.shape[-1] >= 1 << 31:
        raise NativeError(f"{what}: ids {tuple(ids.shape)} and rows of {shape[1]} are too long")
    _ints(ids, device, what, "ids")
    if positions is not None:
        ids, positions = _positions(positions, ids, what)
        if pos_weight is None:
            raise NativeError(f"{what}: positions without a position table")
    if pos_weight is not None:
        if forward_ad._current_level >= 0:
            _no_tangent(pos_weight, what, "pos_weight")
        pshape = pos_weight.shape
        if (len(pshape) != 2 or pshape[1] != shape[1] or pos_weight.dtype != dtype
                or pos_weight.device != device):
            raise NativeError(f"{what}: the position table {tuple(pshape)} {pos_weight.dtype} "
                              f"does not fit {tuple(shape)} {dtype}")
        if positions is None and (ids.ndim < 1 or ids.shape[-1] > pshape[0]):
            raise NativeError(f"{what}: ids {tuple(ids.shape)} have more positions than the "
                              f"table's {pshape[0]}")
    if padding_idx is not None:
        _padding(padding_idx, shape[0], what)
    if out_dtype is not None:
        dtype = out_dtype
        _out_type(dtype, what)
    cut, key = _drop(dropout_p, rng, weight, what)
    if _is_tracing() or torch.is_grad_enabled() and (
            weight.requires_grad or pos_weight is not None and pos_weight.requires_grad):
        return _Embedding.apply(weight, pos_weight, ids, positions, scale, padding_idx,
                                dropout_p, rng, dtype)
    return _embed(ids, weight, pos_weight, positions, scale, cut, key, dtype)


def _padding(padding_idx, rows, what):
    if padding_idx is not None and not 0 <= padding_idx < rows:
        raise NativeError(f"{what}: padding_idx {padding_idx} is not one of {rows} rows")


def _table_grad(given, rows, dtype, grad, what, name):
    """(tensor, add to it) for the gradient of a table."""
    dim = grad.shape[-1]
    if given is None:
        return grad.new_empty((rows, dim), dtype=dtype), False
    _float(given, what, name)
    if given.shape != (rows, dim) or given.device != grad.device or not given.is_contiguous():
        raise NativeError(f"{what}: {name} must be contiguous ({rows}, {dim}) on {grad.device}, "
                          f"got {tuple(given.shape)} on {given.device}")
    return given, True


def embedding_backward(grad, ids, rows, pos_rows=0, positions=None, scale=1.0, padding_idx=None,
                       dropout_p=0.0, rng=None, dtype=torch.float32, weight_grad=None,
                       pos_grad=None):
    """The gradients (rows, dim) and (pos_rows, dim) of embedding's tables from that of its
    result; None for a table of 0 rows.

    Dense, in `dtype`; or added to weight_grad / pos_grad, which are then returned (the
    gradient of a tied head, or that of the micro-batches before).  The sums are fp32, in an
    order that the ids decide: the same inputs give the same bits."""
    what = "embedding_backward"
    _eager(what)
    _float(grad, what, "grad")
    _ints(ids, grad.device, what, "ids")
    if grad.ndim != ids.ndim + 1 or grad.shape[:-1] != ids.shape:
        raise NativeError(f"{what}: grad {tuple(grad.shape)} does not fit ids "
                          f"{tuple(ids.shape)}")
    _out_type(dtype, what)
    if grad.shape[-1] > 1 << 23:
        raise NativeError(f"{what}: rows of {grad.shape[-1]} are too long")
    if rows < 0 or pos_rows < 0:
        raise NativeError(f"{what}: {rows} and {pos_rows} rows")
    _padding(padding_idx, rows, what)
    ids, positions = _positions(positions, ids, what)
    if pos_rows and positions is None and (ids.ndim < 1 or ids.shape[-1] > pos_rows):
        raise NativeError(f"{what}: ids {tuple(ids.shape)} have more positions than {pos_rows}")
    cut, key = _drop(dropout_p, rng, grad, what)
    dim, tokens = grad.shape[-1], ids.numel()
    seq = ids.shape[-1] if ids.ndim else 1
    ids = ids.contiguous()
    grad, _, _, stride = _rows(grad)
    dw = dp = None
    add = pos_add = False
    if rows:
        dw, add = _table_grad(weight_grad, rows, dtype, grad, what, "weight_grad")
    if pos_rows:
        dp, pos_add = _table_grad(pos_grad, pos_rows, dtype, grad, what, "pos_grad")
    padding_idx = -1 if padding_idx is None else padding_idx
    if dw is not None and dp is not None and dw.dtype != dp.dtype:
        # one launch writes one type
        _native.embedding_grad(ids, None, tokens, seq, grad, stride, dim, padding_idx, scale, cut,
                               key, dw, add, None, False)
        _native.embedding_grad(ids, positions, tokens, seq, grad, stride, dim, -1, scale, cut,
                               key, None, False, dp, pos_add)
    elif (rows or pos_rows) and dim:
        _native.embedding_grad(ids, positions, tokens, seq, grad, stride, dim, padding_idx, scale,
                               cut, key, dw, add, dp, pos_add)
    # autograd does not see a write through a pointer
    if add:
        increment_version(dw)
    if pos_add:
        increment_version(dp)
    return dw, dp


# ---- cross entropy --------------------------------------------------------------------------

def _xent_args(logits, targets, label_smoothing, z_loss, reduction, what):
    _float(logits, what, "logits")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise NativeError(f"{what}: logits must be (..., classes), got {tuple(logits.shape)}")
    _ints(targets, logits.device, what, "targets")
    if targets.shape != logits.shape[:-1]:
        raise NativeError(f"{what}: targets {tuple(targets.shape)} do not fit logits "
                          f"{tuple(logits.shape)}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise NativeError(f"{what}: label_smoothing must be between 0 and 1, not "
                          f"{label_smoothing}")
    if not z_loss >= 0.0:
        raise NativeError(f"{what}: z_loss must not be negative, got {z_loss}")
    if reduction not in _REDUCTIONS:
        raise NativeError(f"{what}: reduction {reduction!r} is none of {sorted(_REDUCTIONS)}")


def _xent(logits, rows, targets, ignore_index, smoothing, z_loss, reduction, dlogits=None,
          dstride=0, grad_scale=1.0, keep=False):
    """(loss, statistics for the backward pass if `keep`) and, in place, dlogits; rows:
    _rows(logits)."""
    z, n, classes, stride = rows
    red = _REDUCTIONS[reduction]
    loss = torch.empty(targets.shape if red == 0 else (), dtype=torch.float32,
                       device=logits.device)
    stats = None
    if n or red:
        stats = _native.cross_entropy(z, (n, classes, stride), targets.contiguous(),
                                      ignore_index, smoothing, z_loss, red, grad_scale, loss,
                                      dlogits, dstride, keep)
    return loss, stats


def _like_rows(logits, rows):
    """(tensor, row stride) for the gradient of logits: the rows of a padded view as far apart as
    the view's, which keeps their alignment for this and the next product; else contiguous."""
    z, _, classes, stride = rows
    if z is logits and classes < stride <= classes + 256:
        return torch.empty_strided(logits.shape, logits.stride(), dtype=logits.dtype,
                                   device=logits.device), stride
    return logits.new_empty(logits.shape), classes


def _step_grad(logits, rows, inplace, what):
    """(tensor, row stride) for the gradient of a step: the logits themselves with inplace."""
    z, n, classes, stride = rows
    if not inplace:
        return _like_rows(logits, rows)
    if z is logits and (n <= 1 or stride >= classes):
        return logits, stride
    raise NativeError(f"{what}: logits of strides {tuple(logits.stride())} have no rows to "
                      "write a gradient to")


class _CrossEntropy(Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index, smoothing, z_loss, reduction):
        loss, stats = _xent(logits, _rows(logits), targets, ignore_index, smoothing, z_loss,
                            reduction, keep=True)
        ctx.save_for_backward(logits, targets, stats)
        ctx.args = ignore_index, smoothing, z_loss, _REDUCTIONS[reduction]
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if forward_ad._current_level >= 0:
            _no_tangent(grad, "cross_entropy", "the loss's gradient")
        logits, targets, stats = ctx.saved_tensors
        z, *rows = _rows(logits)
        dz, stride = _like_rows(logits, (z, *rows))
        if dz.numel():
            _native.cross_entropy_grad(z, rows, targets.contiguous(), *ctx.args, stats,
                                       grad.float().contiguous(), dz, stride)
        return dz, *[None] * 5


def cross_entropy(logits, targets, ignore_index=-100, label_smoothing=0.0, z_loss=0.0,
                  reduction="mean"):
    """Cross entropy of logits (..., classes) against integer targets (...), in fp32:

        lse - (1 - s) z_target - s mean(z) + z_loss lse^2,    lse = log sum exp z

    with s the label smoothing; summed, averaged over the rows that have a target, or (for
    "none") one a row.  Rows whose target is ignore_index count for nothing; another target
    outside the classes gives NaN, as does a row of logits that are all -inf."""
    _eager("cross_entropy", function=True)
    _xent_args(logits, targets, label_smoothing, z_loss, reduction, "cross_entropy")
    if _is_tracing() or torch.is_grad_enabled() and logits.requires_grad:
        return _CrossEntropy.apply(logits, targets, ignore_index, label_smoothing, z_loss,
                                   reduction)
    return _xent(logits, _rows(logits), targets, ignore_index, label_smoothing, z_loss,
                 reduction)[0]


def cross_entropy_step(logits, targets, ignore_index=-100, label_smoothing=0.0, z_loss=0.0,
                       reduction="mean", grad_scale=1.0, inplace=False):
    """(loss, dlogits) of cross_entropy ("mean" or "sum") in one pass over the logits, outside
    autograd: each is read once and its gradient written once.

    dlogits is the gradient of grad_scale * loss (1 / micro-batches, a loss scale) in the
    logits' type; with inplace it takes the logits' own memory (what lies beside the rows of a
    padded view stays).  logits.backward(dlogits) goes on from there; after a call in place it
    raises torch's error where the logits' values are needed for it (a soft-cap's tanh, another
    loss of the same logits), and should start at the tensor that the product returned: as for
    any view written in place, autograd copies a view's gradient."""
    what = "cross_entropy_step"
    _eager(what)
    _xent_args(logits, targets, label_smoothing, z_loss, reduction, what)
    logits = logits.detach()
    if reduction == "none":
        raise NativeError(f"{what}: the loss must be a mean or a sum")
    rows = _rows(logits)
    dlogits, dstride = _step_grad(logits, rows, inplace, what)
    loss, _ = _xent(logits, rows, targets, ignore_index, label_smoothing, z_loss, reduction,
                    dlogits, dstride, grad_scale)
    if inplace:   # autograd does not see a write through a pointer
        increment_version(logits)
    return loss, dlogits


# ---- log probabilities ----------------------------------------------------------------------

TokenLogProbs = collections.namedtuple("TokenLogProbs",
                                       "log_probs entropy top_log_probs top_ids")

_MAX_TOP, _MAX_LIST = 256, 1024


def _temperature(tau, what):
    if not isinstance(tau, (int, float)) or not 1e-6 <= tau <= 1e6:
        raise NativeError(f"{what}: temperature must be between 1e-6 and 1e6, not {tau}")


def _log_probs(logits, rows, tokens, top, tau, ignore_index, keep=False):
    """(TokenLogProbs, statistics for the backward pass if `keep`); rows: _rows(logits)."""
    z, n, classes, stride = rows
    shape, device = logits.shape[:-1], logits.device
    entropy = torch.empty(shape, dtype=torch.float32, device=device)
    lp = top_lp = ids = stats = None
    if tokens is not None:
        lp = torch.empty_like(entropy)
        tokens = tokens.contiguous()
    if top:
        top_lp = torch.empty((*shape, top), dtype=torch.float32, device=device)
        ids = torch.empty((*shape, top), dtype=torch.int64, device=device)
    if keep:
        stats = torch.empty(3 * n, dtype=torch.float32, device=device)
    if n:
        _native.log_probs(z, (n, classes, stride), tokens, ignore_index, tau, top, lp, entropy,
                          top_lp, ids, stats)
    return TokenLogProbs(lp, entropy, top_lp, ids), stats


class _TokenLogProbs(Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, tau, ignore_index):
        out, stats = _log_probs(logits, _rows(logits), tokens, top, tau, ignore_index, keep=True)
        ctx.save_for_backward(logits, tokens, out.top_ids, stats)
        ctx.args = tau, ignore_index
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(out.top_ids)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        logits, tokens, ids, stats = ctx.saved_tensors
        tau, ignore_index = ctx.args
        grads = grads[:3]
        if forward_ad._current_level >= 0:
            for g in grads:
                if g is not None:
                    _no_tangent(g, "token_log_probs", "an output's gradient")
        z, *rows = _rows(logits)
        dz, stride = _like_rows(logits, (z, *rows))
        if dz.numel():
            _native.log_probs_grad(
                z, rows, None if tokens is None else tokens.contiguous(), ignore_index, tau, ids,
                stats, [None if g is None else g.float().contiguous() for g in grads], dz, stride)
        return dz, None, None, None, None


def token_log_probs(logits, tokens=None, top=0, temperature=1.0, ignore_index=-100):
    """What logits (..., classes) say, by softmax(logits / temperature), in fp32:

        log_probs      (...)       log probability of each row's token (None without tokens)
        entropy        (...)       of each row
        top_log_probs  (..., top)  the largest log probabilities, falling (None for top 0)
        top_ids        (..., top)  their classes (int64); of equal logits the lower class first

    tokens: int64 or int32 (...); top up to 256.  The three log probabilities and entropies take
    part in autograd.  A row whose token is ignore_index gives zeros, and ignore_index for its
    classes (-100 where that is a class), which distillation leaves out in turn; another token
    outside the classes gives NaN for its log probability (and its row's gradient, if that is
    wanted).  A row without a softmax (a NaN, an infinity, -inf alone) gives NaN, and the classes
    0, 1, ... for its top."""
    what = "token_log_probs"
    _eager(what, function=True)
    _float(logits, what, "logits")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise NativeError(f"{what}: logits must be (..., classes), got {tuple(logits.shape)}")
    if tokens is not None:
        _ints(tokens, logits.device, what, "tokens")
        if tokens.shape != logits.shape[:-1]:
            raise NativeError(f"{what}: tokens {tuple(tokens.shape)} do not fit logits "
                              f"{tuple(logits.shape)}")
    if not isinstance(top, int) or not 0 <= top <= min(_MAX_TOP, logits.shape[-1]):
        raise NativeError(f"{what}: top must be between 0 and {_MAX_TOP} and no more than the "
                          f"{logits.shape[-1]} classes, not {top}")
    _temperature(temperature, what)
    if _is_tracing() or torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, top, temperature,
                                                   ignore_index))
    return _log_probs(logits, _rows(logits), tokens, top, temperature, ignore_index)[0]


# ---- distillation ---------------------------------------------------------------------------

def _distill_args(logits, ids, teacher, tau, reduction, what):
    _float(logits, what, "logits")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise NativeError(f"{what}: logits must be (..., classes), got {tuple(logits.shape)}")
    _ints(ids, logits.device, what, "ids")
    _float(teacher, what, "teacher")
    if (ids.ndim != logits.ndim or ids.shape[:-1] != logits.shape[:-1]
            or teacher.shape != ids.shape or teacher.device != logits.device):
        raise NativeError(f"{what}: ids {tuple(ids.shape)} and teacher {tuple(teacher.shape)} on "
                          f"{teacher.device} do not fit logits {tuple(logits.shape)} on "
                          f"{logits.device}")
    if not 1 <= ids.shape[-1] <= _MAX_LIST:
        raise NativeError(f"{what}: lists must have 1 to {_MAX_LIST} classes, not "
                          f"{ids.shape[-1]}")
    if torch.is_grad_enabled() and teacher.requires_grad:
        raise NativeError(f"{what}: the teacher takes no gradient; give teacher.detach()")
    _temperature(tau, what)
    if reduction not in _REDUCTIONS:
        raise NativeError(f"{what}: reduction {reduction!r} is none of {sorted(_REDUCTIONS)}")


def _distill(logits, rows, ids, teacher, tau, rest, ignore_index, reduction, dlogits=None,
             dstride=0, grad_scale=1.0, keep=False):
    """(loss, statistics for the backward pass if `keep`) and, in place, dlogits; rows:
    _rows(logits)."""
    z, n, classes, stride = rows
    red = _REDUCTIONS[reduction]
    loss = torch.empty(logits.shape[:-1] if red == 0 else (), dtype=torch.float32,
                       device=logits.device)
    stats = None
    if n or red:
        stats = _native.distill(z, (n, classes, stride), ids.contiguous(), teacher.contiguous(),
                                ignore_index, tau, rest, red, grad_scale, loss, dlogits, dstride,
                                keep)
    return loss, stats


class _Distillation(Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, tau, rest, ignore_index, reduction):
        loss, stats = _distill(logits, _rows(logits), ids, teacher, tau, rest, ignore_index,
                               reduction, keep=True)
        ctx.save_for_backward(logits, ids, teacher, stats)
        ctx.args = ignore_index, tau, _REDUCTIONS[reduction]
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if forward_ad._current_level >= 0:
            _no_tangent(grad, "distillation", "the loss's gradient")
        logits, ids, teacher, stats = ctx.saved_tensors
        z, *rows = _rows(logits)
        dz, stride = _like_rows(logits, (z, *rows))
        if dz.numel():
            _native.distill_grad(z, rows, ids.contiguous(), teacher.contiguous(), *ctx.args, stats,
                                 grad.float().contiguous(), dz, stride)
        return dz, *[None] * 6


def distillation(logits, ids, teacher, temperature=1.0, rest=False, ignore_index=-100,
                 reduction="mean"):
    """How far softmax(logits / temperature) is from a teacher's, of which each row has a list of
    classes ids (..., k) with their log probabilities teacher (..., k), in fp32:

        temperature^2 sum over the list of q (log q - log p),    q = softmax(teacher)

    or, with `rest`, q = exp(teacher) and the classes outside the list as one more, whose q is
    what the list's leave of 1 (nothing, if that is within the rounding of their fp32 sum, or if
    there are no logits outside the list but -inf) and whose p is the sum of theirs.  What
    16-bit lists leave by their rounding (of bf16, 2^-8 of each logarithm) is a rest like any
    other: keep lists in fp32 where the student's other classes are masked by finite values, from
    which it would be far.
    Reductions as in cross_entropy, a mean over the rows that have a teacher.

    token_log_probs(teacher_logits, top=k, temperature=temperature) gives such lists: teacher is
    taken as it is, at the temperature already (raw logits go in divided by it, without `rest`).
    k up to 1024; a class named twice counts with both.  The loss carries the rounding of fp32
    logarithms times temperature^2, about 1e-7 of it, and a divergence of zero may come out that far
    below.  An entry whose class is ignore_index is left out, and a row whose first entry is counts
    for nothing.  (An ignore_index that is one of the classes leaves out that class and, as
    token_log_probs marks its lists then, -100.)  Another class outside the logits' makes its row
    NaN, as does a row without a softmax.  An entry of -inf adds nothing, whatever the logits say;
    a row of those alone is NaN, with `rest` it leaves all to the others.  The teacher takes no
    gradient."""
    _eager("distillation", function=True)
    _distill_args(logits, ids, teacher, temperature, reduction, "distillation")
    if _is_tracing() or torch.is_grad_enabled() and logits.requires_grad:
        return _Distillation.apply(logits, ids, teacher, temperature, bool(rest), ignore_index,
                                   reduction)
    return _distill(logits, _rows(logits), ids, teacher, temperature, bool(rest), ignore_index,
                    reduction)[0]


def distillation_step(logits, ids, teacher, temperature=1.0, rest=False, ignore_index=-100,
                      reduction="mean", grad_scale=1.0, inplace=False):
    """(loss, dlogits) of distillation ("mean" or "sum") outside autograd, the logits read once
    where a workgroup's registers hold a row; grad_scale and inplace as in cross_entropy_step."""
    what = "distillation_step"
    _eager(what)
    _distill_args(logits, ids, teacher, temperature, reduction, what)
    logits = logits.detach()
    if reduction == "none":
        raise NativeError(f"{what}: the loss must be a mean or a sum")
    rows = _rows(logits)
    dlogits, dstride = _step_grad(logits, rows, inplace, what)
    loss, _ = _distill(logits, rows, ids, teacher, temperature, bool(rest), ignore_index,
                       reduction, dlogits, dstride, grad_scale)
    if inplace:   # autograd does not see a write through a pointer
        increment_version(logits)
    return loss, dlogits
