"""Layer norm on the library's kernels: `layer_norm` (differentiable) and the module `LayerNorm`.

The reference's models take nn.LayerNorm from torch (its model/model.py blocks); here the norm that
surrounds the library's products is a kernel of the same library. Statistics and sums are fp32
whatever the type of the activations, every result is rounded once, and the reduction of the weight's
and the bias's gradient over the rows has a fixed order: the same call gives the same bits.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib
from ._call import (DTYPE, call, dtype_code, empty, empty_as, empty_rows, once, ptr, refuse_tangents, require_cuda, rows_of,
                    wants_grad)


def _check(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor]) -> None:
    require_cuda(x, weight, bias)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs a last dimension of at least one element")
    dtype_code(x, "x")
    d = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != d:
            raise ValueError(f"{name} must hold one element per column ({d}), got shape {tuple(p.shape)}")
        if p.dtype != x.dtype and p.dtype != torch.float32:
            raise TypeError(f"{name} must be of the type of x ({x.dtype}) or float32, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")


def _dense(p):
    return p if p is None or p.is_contiguous() else p.contiguous()


def _forward(x, weight, bias, eps, stats):
    """(y, statistics): two rows of fp32 values, mean and rstd, or None without ``stats``."""
    xr, rows, ldx = rows_of(x)
    y = empty_as(x)
    w, b = _dense(weight), _dense(bias)
    d = x.shape[-1]
    p = w if w is not None else b
    st, mean, rstd = None, None, None
    if stats:
        st = empty_rows(2, rows, torch.float32, x.device)
        mean = st.data_ptr()
        rstd = mean + 4 * rows
        if rows == 0:
            mean = rstd = None
    code = DTYPE[x.dtype]
    call(x.device, _lib.load().b200s_layer_norm, rows, d, code, code if p is None else DTYPE[p.dtype], eps, xr.data_ptr(), ldx,
         ptr(w), ptr(b), y.data_ptr(), d, mean, rstd)
    return y, st


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows, d):
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().b200s_layer_norm_backward_workspace(rows, d, ctypes.byref(n)))
    return n.value


def _backward(dy, x, weight, st, param_dtype, need_x, need_w, need_b):
    """(dx, dw, db), None where not needed."""
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    xr, rows, ldx = rows_of(x)
    gr, _, ldg = rows_of(dy)
    d, dev = x.shape[-1], x.device
    w = _dense(weight)
    dx = empty_as(x) if need_x else None
    dw = empty(d, param_dtype, dev) if need_w else None
    db = empty(d, param_dtype, dev) if need_b else None
    ws, need = None, 0
    if need_w or need_b:
        need = _workspace_bytes(rows, d)
        ws = empty(need, torch.uint8, dev)     # held until the launch
    mean = st.data_ptr()
    call(dev, _lib.load().b200s_layer_norm_backward, rows, d, DTYPE[x.dtype], DTYPE[param_dtype], xr.data_ptr(), ldx,
         gr.data_ptr(), ldg, ptr(w), mean, mean + 4 * rows, ptr(dx), d, ptr(dw), ptr(db), ptr(ws), need)
    return dx, dw, db


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, st = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, st)
        p = weight if weight is not None else bias
        ctx.param_dtype = x.dtype if p is None else p.dtype
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        x, weight, st = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _backward(dy, x, weight, st, ctx.param_dtype, need[0], need[1], need[2])
        return dx, dw, db, None


# Opaque operators for traced graphs (torch.compile), as for the product (ops.py).
@torch.library.custom_op("b200s::layer_norm", mutates_args=())
def _layer_norm_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
                   eps: float) -> tuple[Tensor, Tensor]:
    return _forward(x, weight, bias, eps, True)


@_layer_norm_op.register_fake
def _(x, weight, bias, eps):
    rows = x.numel() // x.shape[-1]
    return x.new_empty(x.shape), x.new_empty((2, rows), dtype=torch.float32)


@torch.library.custom_op("b200s::layer_norm_backward", mutates_args=())
def _layer_norm_backward_op(dy: Tensor, x: Tensor, weight: Optional[Tensor], st: Tensor,
                            fp32_params: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _backward(dy, x, weight, st, torch.float32 if fp32_params else x.dtype, True, True, True)


@_layer_norm_backward_op.register_fake
def _(dy, x, weight, st, fp32_params):
    pd = torch.float32 if fp32_params else x.dtype
    d = x.shape[-1]
    return x.new_empty(x.shape), x.new_empty((d,), dtype=pd), x.new_empty((d,), dtype=pd)


def _op_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    p = weight if weight is not None else bias
    ctx.fp32_params = p is not None and p.dtype == torch.float32
    ctx.has_bias = bias is not None


def _op_backward(ctx, dy, _dst):
    x, weight, st = ctx.saved_tensors
    dx, dw, db = _layer_norm_backward_op(dy, x, weight, st, ctx.fp32_params)
    return dx, dw if weight is not None else None, db if ctx.has_bias else None, None


_layer_norm_op.register_autograd(_op_backward, setup_context=_op_setup)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """Layer norm of ``x`` over its last dimension, on the current CUDA stream.

    ``weight`` and ``bias`` (one element per column, or None) are of x's type or float32; the result has
    x's type. Rows may be strided (a slice of a wider matrix is not copied). Differentiable in all three
    once; the gradients have the types of their tensors. Nothing is cast under autocast."""
    _check(x, weight, bias)
    if torch.compiler.is_compiling():
        return _layer_norm_op(x, weight, bias, float(eps))[0]
    refuse_tangents(x, weight, bias)
    if wants_grad(x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension (same constructor, parameters and state_dict) on `layer_norm`."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device="cuda", dtype=None) -> None:
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises the last dimension only")

    def forward(self, input: Tensor) -> Tensor:
        if input.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"expected {self.normalized_shape[0]} columns, got shape {tuple(input.shape)}")
        return layer_norm(input, self.weight, self.bias, self.eps)
