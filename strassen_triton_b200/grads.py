"""The global gradient norm over many tensors and clipping to it: `grad_norm`, `clip_grads_` on a list of
gradients, `clip_grad_norm_` on parameters (torch.nn.utils' name and formula).

Two launches for a whole model (more for lists of over 512 tensors), no synchronisation, no copy of the gradients: the
sum of squares (in fp64), then one pass that forms the coefficient on the device and scales. When the
norm is below the bound that pass reads and writes nothing.
"""
from __future__ import annotations

import math
from array import array
from typing import Iterable, Optional, Sequence

import torch
from torch import Tensor

from . import _lib
from ._call import DTYPE, call, empty, require_cuda


def _dense(t: Tensor) -> bool:
    """Do the elements of ``t`` fill one gapless span of memory, each once (in any order)?"""
    if t.is_contiguous():
        return True
    need = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda x: x[1]):
        if size == 1:
            continue
        if stride != need:
            return False
        need *= size
    return True


def _checked(grads: Sequence[Tensor], what: str) -> torch.device:
    """The device of a list of tensors the kernels can take; raises for anything else."""
    if not grads:
        raise ValueError(f"{what} is empty")
    for t in grads:
        require_cuda(grads[0], t)
        if t.dtype not in DTYPE:
            raise TypeError(f"unsupported dtype {t.dtype} in {what} (bfloat16, float16 and float32 are supported)")
        if t.layout is not torch.strided:
            raise TypeError(f"{what} must hold dense tensors")
        if t.numel() and not t.data_ptr():
            raise TypeError(f"{what} holds a {type(t).__name__} without memory of its own (of a sharded tensor pass the "
                            "local part, and the process group)")
    return grads[0].device


def _plain_words(grads):
    """The entries of a list whose tensors are all contiguous, of supported types and on one GPU (what gradients
    nearly always are), one property after the other over the whole list (0.35 us a tensor, 0.6 tensor by tensor);
    None for any other list."""
    if not grads:
        return None
    try:
        devices = set(map(Tensor.get_device, grads))
        if len(devices) != 1 or min(devices) < 0 or not all(map(Tensor.is_contiguous, grads)):
            return None
        types = [t.dtype for t in grads]
        at = list(map(Tensor.data_ptr, grads))          # raises for a tensor that is not dense
        sizes = list(map(Tensor.numel, grads))
    except (AttributeError, RuntimeError, TypeError):
        return None
    if 0 in at and any(n and not p for p, n in zip(at, sizes)):
        return None
    if len(set(types)) == 1:
        code = DTYPE.get(types[0])
        if code is None:
            return None
        words = [code | code << 32] * (4 * len(at))
    else:
        codes = list(map(DTYPE.get, types))
        if None in codes:
            return None
        words = [0] * (4 * len(at))
        words[3::4] = [c | c << 32 for c in codes]
    words[0::4] = words[1::4] = at
    words[2::4] = sizes
    return words


def _entries(src, dst):
    """An array of struct b200s_tensor: four 64-bit words each, the two types in the last."""
    words = []
    for s, d in zip(src, dst):
        words += (s.data_ptr(), d.data_ptr(), s.numel(), DTYPE[s.dtype] | DTYPE[d.dtype] << 32)
    return array("q", words)


def _sumsq(dev, arr, n, group):
    """(parts, how many of them count): the partial sums of squares, of all ranks of ``group`` when given."""
    parts = empty(_lib.NORM_PARTS, torch.float64, dev)
    call(dev, _lib.load().b200s_grad_sumsq, arr.buffer_info()[0], n, parts.data_ptr())
    if group is None:
        return parts, _lib.NORM_PARTS
    import torch.distributed as dist

    total = parts.sum().reshape(1)
    dist.all_reduce(total, group=group)
    return total, 1


def _no_share(device, group, error_if_nonfinite=False) -> Tensor:
    """The norm on a rank that holds no gradient: it still takes its place in the sum over the ranks."""
    import torch.distributed as dist

    total = torch.zeros(1, dtype=torch.float64, device=device)
    dist.all_reduce(total, group=group)
    norm = total.sqrt().float().reshape(())
    if error_if_nonfinite:
        _require_finite(norm)
    return norm


def _require_finite(norm: Tensor) -> None:
    if not math.isfinite(norm.item()):
        raise RuntimeError("the norm of the gradients is not finite, so they cannot be clipped")


def _bound(max_norm) -> float:
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    return max_norm


def grad_norm(grads: Iterable[Tensor], *, group=None) -> Tensor:
    """sqrt of the sum of squares over all tensors, a 0-d float32 tensor, on the current stream. ``group``: a
    process group whose ranks each hold a shard of the gradients; their sums of squares are added (a rank that
    holds none passes an empty list)."""
    grads = list(grads)
    if not grads and group is not None:
        return _no_share(torch.device("cuda", torch.cuda.current_device()), group)
    words = _plain_words(grads)
    if words is not None:
        dev, arr = grads[0].device, array("q", words)
    else:
        dev = _checked(grads, "grads")
        grads = [t if _dense(t) else t.contiguous() for t in grads]
        arr = _entries(grads, grads)
    parts, n_parts = _sumsq(dev, arr, len(grads), group)
    norm = torch.empty_strided((), (), dtype=torch.float32, device=dev)
    call(dev, _lib.load().b200s_grad_norm, parts.data_ptr(), n_parts, norm.data_ptr())
    return norm


@torch.no_grad()
def clip_grads_(grads: Iterable[Tensor], max_norm: float, *, out: Optional[Sequence[Tensor]] = None,
                error_if_nonfinite: bool = False, group=None) -> Tensor:
    """Scale ``grads`` in place by min(1, max_norm / (norm + 1e-6)) and return their norm before that (a 0-d
    float32 tensor, not synchronised).

    ``out``: tensors of the same shapes (any of the supported types, for instance the optimizer's float32
    gradients) that receive the scaled values instead; the gradients are then only read. A norm that is NaN
    makes all results NaN, unless ``error_if_nonfinite`` (which waits for the GPU) raises first. ``group`` as in
    `grad_norm`. A tensor that is written may appear only once and overlap no other one."""
    grads = list(grads)
    max_norm = _bound(max_norm)
    if not grads and group is not None:
        return _no_share(torch.device("cuda", torch.cuda.current_device()), group, error_if_nonfinite)
    words = _plain_words(grads)
    dev = grads[0].device if words is not None else _checked(grads, "grads")
    src, back = grads, []
    if words is None:
        src = [t if _dense(t) else t.contiguous() for t in grads]
    if out is None:
        if words is None:
            for t in grads:
                if any(st == 0 and sz > 1 for sz, st in zip(t.shape, t.stride())):
                    raise ValueError("a gradient with repeated elements (an expanded tensor) cannot be scaled in place")
            back = [(t, s) for t, s in zip(grads, src) if t is not s]
            words = _entries(src, src)
        arr = array("q", words)
    else:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out holds {len(out)} tensors for {len(grads)} gradients")
        quick = _plain_words(out) if words is not None else None
        if quick is None:
            _checked(out, "out")
        if out[0].device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {out[0].device}")
        for i, (t, o) in enumerate(zip(grads, out)):
            if o.shape != t.shape:
                raise ValueError(f"out[{i}] has shape {tuple(o.shape)}, its gradient {tuple(t.shape)}")
        if quick is not None:
            words[1::4] = quick[1::4]
            words[3::4] = [a & 0xffffffff | b & ~0xffffffff for a, b in zip(words[3::4], quick[3::4])]
            arr = array("q", words)
        else:
            src, dst = list(src), []
            for i, o in enumerate(out):
                if o.is_contiguous():
                    src[i] = src[i].contiguous()
                    dst.append(o)
                elif o.stride() == src[i].stride() and _dense(o):
                    dst.append(o)
                else:
                    src[i] = src[i].contiguous()
                    dst.append(torch.empty(o.shape, dtype=o.dtype, device=dev))
                    back.append((o, dst[-1]))
            arr = _entries(src, dst)
    if back:      # the kernels see copies of these, and no overlap
        written = [(t.data_ptr(), t.shape, t.stride()) for t, _ in back if t.numel()]
        if len(set(written)) < len(written):
            raise ValueError("a tensor that is written appears twice in the list")
    lib = _lib.load()
    parts, n_parts = _sumsq(dev, arr, len(grads), group)
    norm = torch.empty_strided((), (), dtype=torch.float32, device=dev)
    if error_if_nonfinite:
        call(dev, lib.b200s_grad_norm, parts.data_ptr(), n_parts, norm.data_ptr())
        _require_finite(norm)
    call(dev, lib.b200s_grad_clip, arr.buffer_info()[0], len(grads), parts.data_ptr(), n_parts, max_norm, norm.data_ptr())
    for t, s in back:
        t.copy_(s)
    # written behind autograd's back: whoever saved one of them for a backward pass learns of it
    torch.autograd.graph.increment_version(grads if out is None else out)
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, *,
                    group=None) -> Tensor:
    """torch.nn.utils.clip_grad_norm_ on the library's kernels: clips the ``grad`` of every parameter (those
    without one are passed over) and returns the norm. Only the 2-norm is offered. ``group`` as in `grad_norm`; a
    rank that has no parameters, or none with a gradient, takes part in the sum."""
    if float(norm_type) != 2.0:
        raise ValueError(f"only norm_type 2 is offered, got {norm_type}")
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    parameters = list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        if group is None:
            return torch.zeros(())
        _bound(max_norm)
        device = parameters[0].device if parameters else torch.device("cuda", torch.cuda.current_device())
        return _no_share(device, group, error_if_nonfinite)
    return clip_grads_(grads, max_norm, error_if_nonfinite=error_if_nonfinite, group=group)
