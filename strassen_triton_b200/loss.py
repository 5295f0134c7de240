"""Log probabilities of given tokens under rows of logits: `token_logprobs` (with the entropy and the most
likely alternatives), and the mean loss `cross_entropy` built on it.

One pass over the logits with a running maximum gives the log-sum-exp and the entropy of a row in fp32;
the backward pass takes the maximum and the log of the sum apart (as one value they would be good to |lse| 2^-24
only), reads the logits once more and writes their gradient. No matrix of probabilities and
no fp32 copy of the logits exists at any time (the reference's training scripts call
F.cross_entropy on logits.float(), which makes both).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _lib
from ._call import call, dtype_code, empty_as, once, ptr, refuse_tangents, require_cuda, rows_of, wants_grad


class TokenLogprobs(NamedTuple):
    logprob: Tensor                  # log probability of every row's target (fp32, targets' shape)
    entropy: Optional[Tensor]        # entropy of every row's distribution (fp32), when asked for
    top_ids: Optional[Tensor]        # (..., top_k) ids of the most likely tokens, best first
    top_logprobs: Optional[Tensor]   # their log probabilities (fp32)


def _forward(logits, targets, vocab, ignore_index, entropy, top_k, stats):
    """(logprob, statistics, entropy, ids, their log probabilities): per row the maximum and the log of the sum, for the
    backward pass, or None without ``stats``."""
    xr, rows, ld = rows_of(logits)
    t = targets.contiguous()
    lp = torch.empty_like(t, dtype=torch.float32)
    ent = torch.empty_like(lp) if entropy else None
    st = lp.new_empty(t.shape + (2,)) if stats else None
    ids = t.new_empty(t.shape + (top_k,)) if top_k else None
    top = torch.empty_like(ids, dtype=torch.float32) if top_k else None
    call(logits.device, _lib.load().b200s_token_logprobs_stats, rows, vocab, dtype_code(logits, "logits"), xr.data_ptr(), ld, t.data_ptr(),
         ignore_index, lp.data_ptr(), ptr(st), ptr(ent), top_k, ptr(ids), ptr(top))
    return lp, st, ent, ids, top


def _backward(logits, targets, vocab, ignore_index, stats, entropy, dlogprob, dentropy):
    xr, rows, ld = rows_of(logits)
    t = targets.contiguous()
    dl, de = (g if g is None or (g.dtype == torch.float32 and g.is_contiguous()) else g.to(torch.float32).contiguous()
              for g in (dlogprob, dentropy))
    out = empty_as(logits)
    width = logits.shape[-1]
    call(logits.device, _lib.load().b200s_token_logprobs_backward_stats, rows, vocab, width, dtype_code(logits, "logits"),
         xr.data_ptr(), ld, t.data_ptr(), ignore_index, stats.data_ptr(), ptr(entropy if de is not None else None),
         ptr(dl), ptr(de), out.data_ptr(), width)
    return out


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, vocab, ignore_index, entropy, top_k):
        lp, st, ent, ids, top = _forward(logits, targets, vocab, ignore_index, entropy, top_k, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, targets, st, ent)
        ctx.cfg = (vocab, ignore_index)
        if top_k:
            ctx.mark_non_differentiable(ids, top)
        return lp, ent, ids, top

    @staticmethod
    @once
    def backward(ctx, dlp, dent, _dids, _dtop):
        logits, targets, st, ent = ctx.saved_tensors
        if dlp is None and dent is None:
            return None, None, None, None, None, None
        return _backward(logits, targets, *ctx.cfg, st, ent, dlp, dent), None, None, None, None, None


# Opaque operators for traced graphs (torch.compile). Outputs that were not asked for are empty.
@torch.library.custom_op("b200s::token_logprobs", mutates_args=())
def _logprobs_op(logits: Tensor, targets: Tensor, vocab: int, ignore_index: int, entropy: bool,
                 top_k: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    lp, st, ent, ids, top = _forward(logits, targets, vocab, ignore_index, entropy, top_k, True)
    e = lambda dt: torch.empty(0, dtype=dt, device=logits.device)  # noqa: E731
    return (lp, st, e(torch.float32) if ent is None else ent, e(torch.int64) if ids is None else ids,
            e(torch.float32) if top is None else top)


@_logprobs_op.register_fake
def _(logits, targets, vocab, ignore_index, entropy, top_k):
    f = lambda *s: logits.new_empty(s, dtype=torch.float32)  # noqa: E731
    shape = tuple(targets.shape)
    tops = shape + (top_k,) if top_k else (0,)
    return (f(*shape), f(*shape, 2), f(*(shape if entropy else (0,))), logits.new_empty(tops, dtype=torch.int64), f(*tops))


@torch.library.custom_op("b200s::token_logprobs_backward", mutates_args=())
def _logprobs_backward_op(logits: Tensor, targets: Tensor, vocab: int, ignore_index: int, stats: Tensor,
                          entropy: Optional[Tensor], dlogprob: Optional[Tensor], dentropy: Optional[Tensor]) -> Tensor:
    return _backward(logits, targets, vocab, ignore_index, stats, entropy, dlogprob, dentropy)


@_logprobs_backward_op.register_fake
def _(logits, targets, vocab, ignore_index, stats, entropy, dlogprob, dentropy):
    return logits.new_empty(logits.shape)


def _op_setup(ctx, inputs, output):
    logits, targets, vocab, ignore_index, entropy, _ = inputs
    _, st, ent, _, _ = output
    ctx.save_for_backward(logits, targets, st, ent)
    ctx.cfg = (vocab, ignore_index, entropy)
    ctx.set_materialize_grads(False)


def _op_backward(ctx, dlp, _dstats, dent, _dids, _dtop):
    logits, targets, st, ent = ctx.saved_tensors
    vocab, ignore_index, has_ent = ctx.cfg
    if dlp is None and (dent is None or not has_ent):
        return None, None, None, None, None, None
    g = _logprobs_backward_op(logits, targets, vocab, ignore_index, st, ent if has_ent else None, dlp,
                              dent if has_ent else None)
    return g, None, None, None, None, None


_logprobs_op.register_autograd(_op_backward, setup_context=_op_setup)


def token_logprobs(logits: Tensor, targets: Tensor, *, vocab: Optional[int] = None, ignore_index: int = -100,
                   entropy: bool = False, top_k: int = 0) -> TokenLogprobs:
    """Log probability of ``targets[...]`` under ``softmax(logits[..., :vocab])``, on the current CUDA stream.

    logits: (..., width) of bfloat16, float16 or float32, rows may be strided; targets: (...) of int64 (int32
    is converted). Columns from ``vocab`` on are padding: never a target or an alternative, gradient zero.
    A target equal to ``ignore_index`` gives 0 and no gradient; any other outside [0, vocab) gives NaN.
    -inf logits are forbidden tokens; a row of nothing else gives -inf, entropy 0 and no gradient.
    ``entropy`` adds the entropy of every row (its gradient also reaches ignored rows), ``top_k`` (at most 64)
    the most likely tokens, ties in favour of the lower id. logprob and entropy are differentiable once."""
    require_cuda(logits, targets)
    dtype_code(logits, "logits")
    if logits.dim() < 1 or logits.shape[:-1] != targets.shape:
        raise ValueError(f"targets must have the shape of logits without its last dimension, got {tuple(targets.shape)} "
                         f"for {tuple(logits.shape)}")
    if targets.dtype == torch.int32:
        targets = targets.long()
    elif targets.dtype != torch.int64:
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    width = logits.shape[-1]
    vocab = width if vocab is None else int(vocab)
    if not 0 < vocab <= width:
        raise ValueError(f"vocab must be within 1 .. {width}, got {vocab}")
    top_k = int(top_k)
    if not 0 <= top_k <= min(vocab, _lib.MAX_TOP_K):
        raise ValueError(f"top_k must be within 0 .. {min(vocab, _lib.MAX_TOP_K)}, got {top_k}")
    ignore_index = int(ignore_index)
    if torch.compiler.is_compiling():
        lp, _, ent, ids, top = _logprobs_op(logits, targets, vocab, ignore_index, bool(entropy), top_k)
        return TokenLogprobs(lp, ent if entropy else None, ids if top_k else None, top if top_k else None)
    refuse_tangents(logits)
    if wants_grad(logits):
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, targets, vocab, ignore_index, bool(entropy), top_k))
    lp, _, ent, ids, top = _forward(logits, targets, vocab, ignore_index, bool(entropy), top_k, False)
    return TokenLogprobs(lp, ent, ids, top)


def cross_entropy(logits: Tensor, targets: Tensor, *, vocab: Optional[int] = None, ignore_index: int = -100,
                  reduction: str = "mean") -> Tensor:
    """The loss -logprob of every target, its sum, or its mean over the targets that are not ignored (NaN when
    all are), as F.cross_entropy with class indices; fp32."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    lp = token_logprobs(logits, targets, vocab=vocab, ignore_index=ignore_index).logprob
    if reduction == "none":
        return -lp
    if reduction == "sum":
        return -lp.sum()
    return -lp.sum() / (targets != ignore_index).sum()
