"""What the tensor-level operators share: argument checks, rows of a tensor, calls on a tensor's device."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPE = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}


def dtype_code(t: torch.Tensor, what: str) -> int:
    code = DTYPE.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {t.dtype} of {what} (bfloat16, float16 and float32 are supported)")
    return code


def require_cuda(first: torch.Tensor, *others) -> None:
    """All of them (None aside) CUDA tensors of one device."""
    try:
        index = first.get_device()
        if index >= 0:
            for t in others:
                if t is not None and t.get_device() != index:
                    break
            else:
                return
    except AttributeError:
        pass
    for t in (first,) + others:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"expected a torch.Tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError("b200s kernels run on CUDA tensors only; there is no CPU path "
                               f"(got a tensor on {t.device})")
        if t.device != first.device:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


def ptr(t):
    return None if t is None else t.data_ptr()


def empty(n: int, dtype, device) -> torch.Tensor:
    """torch.empty(n) (an allocation with its strides given costs 1.5 us, one without 2.3)."""
    return torch.empty_strided((n,), (1,), dtype=dtype, device=device)


def empty_rows(rows: int, cols: int, dtype, device) -> torch.Tensor:
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def empty_as(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def call(device: torch.device, fn, *args) -> None:
    """fn(*args, stream) on the current stream of ``device``; a negative status raises."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def rows_of(t: torch.Tensor):
    """(tensor, rows, row stride) of ``t`` as a matrix of rows along its last dimension; a view wherever
    the strides allow one, a copy otherwise."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, (t.numel() // d if d else 0), d
    m = t.reshape(-1, d) if t.dim() != 2 else t
    if (m.stride(1) != 1 and d > 1) or m.stride(0) < 0:
        m = m.contiguous()
    return m, m.shape[0], m.stride(0)


def once(backward):
    """once_differentiable for an autograd function's backward, without its bookkeeping in the usual case that no
    graph of the backward pass is being recorded."""
    slow = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return slow(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def refuse_tangents(*tensors) -> None:
    """The operators have no forward-mode derivative: a dual tensor's would be lost in silence."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("this operator has no forward-mode derivative (got a dual tensor)")


def wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False
