"""Tensor-level entry to libb200s.so: `matmul(A, B, ...)` on CUDA tensors, and the autograd
function every reference-named module in this repository routes through.

torch is plumbing here (device memory, streams, autograd bookkeeping); all arithmetic runs in
the CUDA library through its C ABI.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Optional

import torch

from . import _call, _lib

_DTYPE = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
_ALGO = {"auto": _lib.ALGO_AUTO, "dense": _lib.ALGO_DENSE, "classic": _lib.ALGO_CLASSIC,
         "strassen": _lib.ALGO_CLASSIC, "winograd": _lib.ALGO_WINOGRAD}


def resolve_precision(precision):
    """How fp32 operands reach the tensor cores: "tf32" (one pass) or "3xtf32" (hi/lo split, three
    passes, fp32-level accuracy). ``None`` follows ``torch.backends.cuda.matmul.allow_tf32``, the
    switch the reference's scripts set (main_profiling.py:31-34): TF32 when it is on, else the
    three-pass mode, as torch.mm would then compute in full fp32."""
    if precision is None:
        return "tf32" if torch.backends.cuda.matmul.allow_tf32 else "3xtf32"
    if precision not in ("tf32", "3xtf32"):
        raise ValueError("precision must be 'tf32', '3xtf32' or None")
    return precision


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"expected a torch.Tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError("b200s kernels run on CUDA tensors only; there is no CPU path "
                               f"(got a tensor on {t.device})")


def _operand(t: torch.Tensor):
    """(tensor, major_is_inner, ld, batch_stride) for a 2-D or 3-D operand, copying only when
    neither of the last two dimensions has unit stride or the strides break 16-byte alignment."""
    es = t.element_size()

    def ok(x):
        r, c = x.shape[-2], x.shape[-1]
        sr, sc = x.stride(-2), x.stride(-1)
        bs = x.stride(0) if x.dim() == 3 else 0
        if (x.data_ptr() % 16) or (bs * es) % 16:
            return None
        if sc == 1 and (sr * es) % 16 == 0 and sr >= c:
            return (True, sr, bs)       # rows x cols with cols contiguous
        if sr == 1 and (sc * es) % 16 == 0 and sc >= r:
            return (False, sc, bs)      # columns contiguous: a transposed view
        return None

    got = ok(t)
    if got is None:
        t = t.contiguous()
        got = ok(t)
        if got is None:
            raise ValueError("operand rows must be a multiple of 16 bytes long "
                             f"(shape {tuple(t.shape)}, dtype {t.dtype})")
    return (t,) + got


def make_problem(A, B, C, algo="auto", depth=-1, beta=0, prod_dtype=None, precision=None,
                 tile_variant=0, pipeline=0, b_blocks_ready=False, fuse=0):
    """Fill a ``b200s_problem`` for C (+)= A @ B. Returns (problem, A', B') where A'/B' are the
    tensors whose pointers must be passed (copies only when the strides force one)."""
    if A.dim() != B.dim() or A.dim() not in (2, 3):
        raise ValueError("A and B must both be 2-D, or both 3-D (batched)")
    if A.dtype != B.dtype or A.dtype not in _DTYPE:
        raise TypeError(f"unsupported operand dtypes {A.dtype}, {B.dtype}")
    if C.dtype not in _DTYPE:
        raise TypeError(f"unsupported output dtype {C.dtype}")
    M, K = A.shape[-2], A.shape[-1]
    K2, N = B.shape[-2], B.shape[-1]
    assert K == K2 and C.shape[-2] == M and C.shape[-1] == N, "shape mismatch"
    batch = A.shape[0] if A.dim() == 3 else 1
    if A.dim() == 3:
        assert B.shape[0] == batch and C.shape[0] == batch, "batch mismatch"
    if C.stride(-1) != 1:
        raise ValueError("C must be row-major (unit stride in its last dimension)")
    A2, a_inner, lda, sa = _operand(A)
    B2, b_inner, ldb, sb = _operand(B)
    p = _lib.Problem()
    p.M, p.N, p.K, p.batch = M, N, K, batch
    p.lda, p.ldb, p.ldc = lda, ldb, C.stride(-2)
    p.strideA, p.strideB = sa, sb
    p.strideC = C.stride(0) if C.dim() == 3 else 0
    # A is M x K: inner-contiguous means K-major. B is K x N: inner-contiguous means N-major.
    p.a_major = _lib.K_MAJOR if a_inner else _lib.MN_MAJOR
    p.b_major = _lib.MN_MAJOR if b_inner else _lib.K_MAJOR
    p.in_dtype = _DTYPE[A.dtype]
    p.out_dtype = _DTYPE[C.dtype]
    p.algo = _ALGO[algo] if isinstance(algo, str) else int(algo)
    p.depth = int(depth)
    p.beta = int(beta)
    p.prod_dtype = -1 if prod_dtype is None else _DTYPE[prod_dtype]
    p.precision = _lib.PREC_3XTF32 if resolve_precision(precision) == "3xtf32" else _lib.PREC_TF32
    p.tile_variant = int(tile_variant)
    p.pipeline = int(pipeline)
    p.b_blocks_ready = 1 if b_blocks_ready else 0
    p.fuse = int(fuse)
    return p, A2, B2


def workspace_bytes(p: "_lib.Problem") -> int:
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().b200s_workspace_bytes(ctypes.byref(p), ctypes.byref(n)))
    return n.value


def resolve(p: "_lib.Problem"):
    a, d = ctypes.c_int32(0), ctypes.c_int32(0)
    _lib.check(_lib.load().b200s_resolve(ctypes.byref(p), ctypes.byref(a), ctypes.byref(d)))
    return a.value, d.value


def matmul_out(A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *, algo="auto", depth=-1, beta=0,
               prod_dtype=None, precision=None, tile_variant=0, pipeline=0, b_blocks_ready=False, fuse=0,
               workspace: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """C = A @ B (beta=0) or C += A @ B (beta=1) on the current CUDA stream, plus ``bias`` (N elements
    of C's dtype, added to every row before the rounding) when given. Returns C."""
    _require_cuda(A, B, C)
    if bias is not None:
        _require_cuda(bias)
        if bias.dim() != 1 or bias.shape[0] != B.shape[-1] or A.dim() != 2:
            raise ValueError("bias must hold one element per column of a 2-D product")
        bias = bias.to(C.dtype).contiguous()
    lib = _lib.load()
    p, A2, B2 = make_problem(A, B, C, algo, depth, beta, prod_dtype, precision, tile_variant, pipeline, b_blocks_ready,
                             fuse)
    with torch.cuda.device(C.device):
        need = workspace_bytes(p)
        ws_ptr = None
        if need:
            if workspace is None or workspace.numel() * workspace.element_size() < need:
                workspace = torch.empty(need, dtype=torch.uint8, device=C.device)
            ws_ptr = workspace.data_ptr()
        stream = torch.cuda.current_stream(C.device).cuda_stream
        if bias is None:
            rc = lib.b200s_matmul(ctypes.byref(p), A2.data_ptr(), B2.data_ptr(), C.data_ptr(), ws_ptr,
                                  need if need else 0, stream)
        else:
            rc = lib.b200s_matmul_bias(ctypes.byref(p), A2.data_ptr(), B2.data_ptr(), bias.data_ptr(), C.data_ptr(),
                                       ws_ptr, need if need else 0, stream)
        _lib.check(rc)
        if workspace is not None:
            workspace.record_stream(torch.cuda.current_stream(C.device))
    return C


def matmul(A: torch.Tensor, B: torch.Tensor, *, algo="auto", depth=-1, out_dtype=None, prod_dtype=None,
           precision=None, tile_variant=0, pipeline=0, b_blocks_ready=False, fuse=0, workspace=None,
           bias=None) -> torch.Tensor:
    """A @ B (+ bias) as a new tensor of ``out_dtype`` (default: the operand dtype)."""
    _require_cuda(A, B)
    shape = (A.shape[-2], B.shape[-1]) if A.dim() == 2 else (A.shape[0], A.shape[-2], B.shape[-1])
    C = torch.empty(shape, dtype=out_dtype or A.dtype, device=A.device)
    return matmul_out(A, B, C, algo=algo, depth=depth, beta=0, prod_dtype=prod_dtype, precision=precision,
                      tile_variant=tile_variant, pipeline=pipeline, b_blocks_ready=b_blocks_ready, fuse=fuse,
                      workspace=workspace, bias=bias)


def device_status(device=None):
    """(status, detail) of the device status word; synchronises the current stream."""
    lib = _lib.load()
    s, d = ctypes.c_int32(0), ctypes.c_int32(0)
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        stream = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.b200s_device_status(stream, ctypes.byref(s), ctypes.byref(d)))
    return s.value, d.value


STAGES = ("operand_blocks_A", "operand_blocks_B", "products", "recombination")


@contextlib.contextmanager
def stage_timing(max_calls: int = 256):
    """Collect the library's per-stage event timing for the matmul calls made inside the block.
    Yields a dict that, after the block, holds the mean milliseconds of the four stages (keys
    ``STAGES``; in the fused schedule: the first group's blocks of A and of B, the fused kernel, the
    recombination left after it) and ``calls``, the number of calls measured."""
    lib = _lib.load()
    _lib.check(lib.b200s_profile_begin(int(max_calls)))
    out = {}
    try:
        yield out
    finally:
        ms = (ctypes.c_float * 4)()
        calls = ctypes.c_int32(0)
        _lib.check(lib.b200s_profile_end(ms, ctypes.byref(calls)))
        out.update({k: float(ms[i]) for i, k in enumerate(STAGES)})
        out["calls"] = calls.value


# ---- the differentiable product as a torch.library custom op ------------------------------------
# The reference wraps its layers and whole models in torch.compile (main_profiling.py:130-144,
# modded_nanogpt/data_dist_train_gpt2.py:721); its own matmuls are plain torch ops that dynamo traces
# through. A ctypes call cannot be traced, so the product is registered as an opaque operator with a
# shape-only (fake) implementation and an autograd formula: dynamo and AOT autograd then carry it
# through a compiled graph without a graph break, forward and backward.
_DT_NAME = {None: "", torch.bfloat16: "bf16", torch.float16: "fp16", torch.float32: "fp32"}
_NAME_DT = {v: k for k, v in _DT_NAME.items()}


@torch.library.custom_op("b200s::matmul", mutates_args=())
def _matmul_op(X: torch.Tensor, W: torch.Tensor, algo: str, depth: int, prod_dtype: str) -> torch.Tensor:
    return matmul(X, W, algo=algo, depth=depth, prod_dtype=_NAME_DT[prod_dtype])


@_matmul_op.register_fake
def _(X, W, algo, depth, prod_dtype):
    shape = (X.shape[-2], W.shape[-1]) if X.dim() == 2 else (X.shape[0], X.shape[-2], W.shape[-1])
    return X.new_empty(shape)


def _matmul_setup(ctx, inputs, output):
    X, W, algo, depth, prod_dtype = inputs
    ctx.save_for_backward(X, W)
    ctx.cfg = (algo, depth, prod_dtype)


def _matmul_backward(ctx, dY):
    """dX = dY @ W^T and dW = X^T @ dY through the same operator, with transposed views (no copies).
    The reference has no custom backward: autograd differentiates its slice/add/mm graph
    (fixed_strassen_fp32_agg.py:13-125), which computes these same two products."""
    X, W = ctx.saved_tensors
    algo, depth, prod_dtype = ctx.cfg
    dX = dW = None
    if dY.dtype != X.dtype:
        dY = dY.to(X.dtype)
    if ctx.needs_input_grad[0]:
        dX = _matmul_op(dY, W.transpose(-1, -2), algo, depth, prod_dtype)
    if ctx.needs_input_grad[1]:
        dW = _matmul_op(X.transpose(-1, -2), dY, algo, depth, prod_dtype)
    return dX, dW, None, None, None


_matmul_op.register_autograd(_matmul_backward, setup_context=_matmul_setup)


@torch.library.custom_op("b200s::linear", mutates_args=())
def _linear_op(X: torch.Tensor, W: torch.Tensor, bias: torch.Tensor, algo: str, depth: int) -> torch.Tensor:
    """X @ W + bias with the bias added in the product's epilogue (X 2-D, W given as weight.T)."""
    if depth > 2:      # the recursion above two levels has no epilogue of its own to carry the bias
        return matmul(X, W, algo=algo, depth=depth) + bias.to(X.dtype)
    return matmul(X, W, algo=algo, depth=depth, bias=bias)


@_linear_op.register_fake
def _(X, W, bias, algo, depth):
    return X.new_empty((X.shape[0], W.shape[1]))


def _linear_setup(ctx, inputs, output):
    X, W, bias, algo, depth = inputs
    ctx.save_for_backward(X, W)
    ctx.cfg = (algo, depth, bias.dtype)


def _linear_backward(ctx, dY):
    X, W = ctx.saved_tensors
    algo, depth, bias_dtype = ctx.cfg
    dX = dW = db = None
    if ctx.needs_input_grad[2]:
        db = dY.sum(0).to(bias_dtype)
    if dY.dtype != X.dtype:
        dY = dY.to(X.dtype)
    if ctx.needs_input_grad[0]:
        dX = _matmul_op(dY, W.transpose(-1, -2), algo, depth, "")
    if ctx.needs_input_grad[1]:
        dW = _matmul_op(X.transpose(-1, -2), dY, algo, depth, "")
    return dX, dW, db, None, None


_linear_op.register_autograd(_linear_backward, setup_context=_linear_setup)


def linear_autograd(X, W, bias, algo="auto", depth=-1):
    """Differentiable X @ W + bias (X 2-D, W = weight.T as a view), the bias fused into the epilogue."""
    _require_cuda(X, W, bias)
    if not torch.compiler.is_compiling():
        _call.refuse_tangents(X, W, bias)
    return _linear_op(X, W, bias, algo, int(depth))


def matmul_autograd(X, W, algo="auto", depth=-1, prod_dtype=None):
    """Differentiable X @ W (2-D or batched 3-D operands); traceable by torch.compile."""
    _require_cuda(X, W)
    if not torch.compiler.is_compiling():
        _call.refuse_tangents(X, W)
    return _matmul_op(X, W, algo, int(depth), _DT_NAME[prod_dtype])


# ---- linear layer with bias, activation and residual in the product's epilogue --------------------
ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "relu2": _lib.ACT_RELU2, "silu": _lib.ACT_SILU,
               "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH}


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """A 2-D operand whose rows (or columns) TMA can address: ``t`` itself, or a copy with its rows padded
    to whole 16-byte vectors. The padding is never read: the product's extents stay those of ``t``."""
    es = t.element_size()
    sr, sc = t.stride()
    if t.data_ptr() % 16 == 0:
        if sc == 1 and sr >= t.shape[1] and sr * es % 16 == 0:
            return t
        if sr == 1 and sc >= t.shape[0] and sc * es % 16 == 0:
            return t
    if sr == 1 and sc > 1:
        return _aligned(t.t()).t()
    v = 16 // es
    out = torch.empty((t.shape[0], (t.shape[1] + v - 1) // v * v), dtype=t.dtype, device=t.device)[:, :t.shape[1]]
    return out.copy_(t)


def _split_k(t: torch.Tensor, dim: int) -> torch.Tensor:
    """fp32 operands run as three TF32 passes over K segments of whole 16-byte vectors: zeros up to those."""
    if t.dtype != torch.float32 or t.shape[dim] % 4 == 0:
        return t
    pad = -t.shape[dim] % 4
    return torch.nn.functional.pad(t, (0, pad) if dim == 1 else (0, 0, 0, pad))


def _epilogue_product(A, B, C, activation, bias, residual, preact, algo, depth, precision):
    """C = act(A @ B + bias) + residual on 2-D operands, z into ``preact`` when given."""
    A, B = _aligned(_split_k(A, 1)), _aligned(_split_k(B, 0))
    p, A, B = make_problem(A, B, C, algo, depth, 0, None, precision)
    e = _lib.Epilogue()
    e.activation = activation
    if bias is not None:
        e.bias = bias.data_ptr()
    if residual is not None:
        e.residual, e.ld_residual = residual.data_ptr(), residual.stride(0)
    if preact is not None:
        e.preact, e.ld_preact = preact.data_ptr(), preact.stride(0)
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    pp, pe = ctypes.byref(p), ctypes.byref(e)
    rc = lib.b200s_matmul_epilogue_workspace(pp, pe, ctypes.byref(n))
    if rc:
        _lib.check(rc)
    ws = torch.empty(n.value, dtype=torch.uint8, device=C.device) if n.value else None
    _call.call(C.device, lib.b200s_matmul_epilogue, pp, pe, A.data_ptr(), B.data_ptr(), C.data_ptr(),
               ws.data_ptr() if ws is not None else None, n.value)
    return C


def _linear_act_forward(x, weight, bias, residual, act, algo, depth, precision, save):
    """(y, z) of 2-D x; z (what the backward pass needs of the pre-activation) is None for "none" or without
    ``save``."""
    M, N = x.shape[0], weight.shape[0]
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    z = torch.empty((M, N), dtype=x.dtype, device=x.device) if save and act != _lib.ACT_NONE else None
    if M:
        r = residual
        if r is not None and ((r.stride(1) != 1 and N > 1) or r.stride(0) < 0):
            r = r.contiguous()
        _epilogue_product(x, weight.t(), y, act, bias, r, z, algo, depth, precision)
    return y, z


def _linear_act_backward(dy, x, weight, z, act, algo, depth, precision, need_x, need_w, need_b):
    """(dx, dw, db) of 2-D dy and x, None where not needed."""
    M, N = dy.shape
    K = x.shape[1]
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    if M == 0:
        return (torch.empty_like(x) if need_x else None, torch.zeros_like(weight) if need_w else None,
                weight.new_zeros(N) if need_b else None)
    if (dy.stride(1) != 1 and N > 1) or dy.stride(0) < 0:
        dy = dy.contiguous()
    lib, dev = _lib.load(), x.device
    dz, db = dy, None
    products = need_x or need_w
    if act != _lib.ACT_NONE or need_b:
        out = None
        if act != _lib.ACT_NONE and products:
            v = 16 // x.element_size()
            out = torch.empty((M, (N + v - 1) // v * v), dtype=x.dtype, device=dev)[:, :N]
            dz = out
        ws, need = None, 0
        if need_b:
            db = torch.empty(N, dtype=x.dtype, device=dev)
            n = ctypes.c_size_t(0)
            _lib.check(lib.b200s_epilogue_backward_workspace(M, N, ctypes.byref(n)))
            need = n.value
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        if out is not None or db is not None:
            _call.call(dev, lib.b200s_epilogue_backward, M, N, _DTYPE[x.dtype], act, _call.ptr(z),
                       z.stride(0) if z is not None else 0, dy.data_ptr(), dy.stride(0), _call.ptr(out),
                       out.stride(0) if out is not None else 0, _call.ptr(db), _call.ptr(ws), need)
    dx = dw = None
    if products:
        dz = _aligned(dz)
    if need_x:
        dx = torch.empty((M, K), dtype=x.dtype, device=dev)
        _epilogue_product(dz, weight, dx, _lib.ACT_NONE, None, None, None, algo, depth, precision)
    if need_w:
        dw = torch.empty((N, K), dtype=x.dtype, device=dev)
        _epilogue_product(dz.t(), x, dw, _lib.ACT_NONE, None, None, None, algo, depth, precision)
    return dx, dw, db


# The dense layer of 16-bit operands with contiguous rows: one call of the library each way.
@functools.lru_cache(maxsize=1024)
def _dense_workspace(backward, M, N, K, code, act, copies):
    n = ctypes.c_size_t(0)
    lib = _lib.load()
    if backward:
        _lib.check(lib.b200s_linear_act_backward_workspace(M, N, K, code, act, copies, ctypes.byref(n)))
    else:
        _lib.check(lib.b200s_linear_act_workspace(M, N, K, code, copies, ctypes.byref(n)))
    return n.value


def _off_grid(t) -> bool:
    """Does TMA need a copy of these rows?"""
    return t.data_ptr() % 16 != 0 or t.stride(0) % 8 != 0 or t.stride(0) < t.shape[1]


def _rows_contiguous(t) -> bool:
    return (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= 0


def _dense_forward(x, weight, bias, residual, act, save):
    """(y, z): z has its rows padded to whole 16-byte vectors, None when the backward pass needs none."""
    M, K = x.shape
    N, dt, dev = weight.shape[0], x.dtype, x.device
    y = _call.empty_rows(M, N, dt, dev)
    z, ldz = None, 0
    if save and act:
        ldz = (N + 7) // 8 * 8
        z = _call.empty_rows(M, ldz, dt, dev)
    rp, ldr = None, 0
    if residual is not None:
        if not _rows_contiguous(residual):
            residual = residual.contiguous()
        rp, ldr = residual.data_ptr(), residual.stride(0)
    code = _DTYPE[dt]
    need = _dense_workspace(False, M, N, K, code, 0, 1 if _off_grid(x) or _off_grid(weight) else 0)
    # held until the launch: freed, it could go to another thread's call on this stream before that
    ws = _call.empty(need, torch.uint8, dev) if need else None
    _call.call(dev, _lib.load().b200s_linear_act, M, N, K, code, act, x.data_ptr(), x.stride(0), weight.data_ptr(),
               weight.stride(0), None if bias is None else bias.data_ptr(), rp, ldr, y.data_ptr(), N,
               None if z is None else z.data_ptr(), ldz, None if ws is None else ws.data_ptr(), need)
    return y, z


def _dense_backward(dy, x, weight, z, act, need_x, need_w, need_b):
    M, K = x.shape
    N, dt, dev = weight.shape[0], x.dtype, x.device
    if dy.dtype != dt:
        dy = dy.to(dt)
    if not _rows_contiguous(dy):
        dy = dy.contiguous()
    dx = _call.empty_rows(M, K, dt, dev) if need_x else None
    dw = _call.empty_rows(N, K, dt, dev) if need_w else None
    db = _call.empty(N, dt, dev) if need_b else None
    code = _DTYPE[dt]
    need = _dense_workspace(True, M, N, K, code, act, 1 if _off_grid(x) or _off_grid(weight) or _off_grid(dy) else 0)
    ws = _call.empty(need, torch.uint8, dev)
    p = _call.ptr
    _call.call(dev, _lib.load().b200s_linear_act_backward, M, N, K, code, act, x.data_ptr(), x.stride(0), weight.data_ptr(),
               weight.stride(0), p(z), z.shape[1] if z is not None else 0, dy.data_ptr(), dy.stride(0), p(dx), K, p(dw), K,
               p(db), ws.data_ptr(), need)
    return dx, dw, db


def _auto_is_dense(M, N, K, code) -> bool:
    """Does the tuner table choose the dense product for the layer and for both products of its backward pass?"""
    lookup = _lib.load().b200s_tuner_lookup
    a, d = ctypes.c_int32(0), ctypes.c_int32(0)
    pa, pd = ctypes.byref(a), ctypes.byref(d)
    for m, n, k in ((M, N, K), (M, K, N), (N, K, M)):
        if lookup(m, n, k, code, pa, pd) or (a.value != _lib.ALGO_DENSE and d.value != 0):
            return False
    return True


class _DenseLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        need = ctx.needs_input_grad
        y, z = _dense_forward(x, weight, bias, residual, act, need[0] or need[1] or need[2])
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        return y

    @staticmethod
    @_call.once
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            x, weight, z = ctx.saved_tensors
            dx, dw, db = _dense_backward(dy, x, weight, z, ctx.act, need[0], need[1], need[2])
        return dx, dw, db, dy if need[3] else None, None


class _LinearActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, algo, depth, precision):
        need = ctx.needs_input_grad
        y, z = _linear_act_forward(x, weight, bias, residual, act, algo, depth, precision, any(need[:3]))
        ctx.save_for_backward(x, weight, z)
        ctx.cfg = (act, algo, depth, precision)
        return y

    @staticmethod
    @_call.once
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = _linear_act_backward(dy, x, weight, z, *ctx.cfg, *need[:3])
        return dx, dw, db, dy if need[3] else None, None, None, None, None


@torch.library.custom_op("b200s::linear_act", mutates_args=())
def _linear_act_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                   residual: Optional[torch.Tensor], act: int, algo: str, depth: int,
                   precision: str) -> tuple[torch.Tensor, torch.Tensor]:
    y, z = _linear_act_forward(x, weight, bias, residual, act, algo, depth, precision or None, True)
    return y, (x.new_empty(0) if z is None else z)


@_linear_act_op.register_fake
def _(x, weight, bias, residual, act, algo, depth, precision):
    shape = (x.shape[0], weight.shape[0])
    return x.new_empty(shape), x.new_empty(shape if act != _lib.ACT_NONE else (0,))


@torch.library.custom_op("b200s::linear_act_backward", mutates_args=())
def _linear_act_backward_op(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, z: torch.Tensor, act: int,
                            algo: str, depth: int, precision: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _linear_act_backward(dy, x, weight, z if act != _lib.ACT_NONE else None, act, algo, depth, precision or None,
                                True, True, True)


@_linear_act_backward_op.register_fake
def _(dy, x, weight, z, act, algo, depth, precision):
    return x.new_empty(x.shape), weight.new_empty(weight.shape), weight.new_empty((weight.shape[0],))


def _linear_act_setup(ctx, inputs, output):
    x, weight, bias, residual, act, algo, depth, precision = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.cfg = (act, algo, depth, precision)
    ctx.has = (bias is not None, residual is not None)


def _linear_act_op_backward(ctx, dy, _dz):
    x, weight, z = ctx.saved_tensors
    dx, dw, db = _linear_act_backward_op(dy, x, weight, z, *ctx.cfg)
    return dx, dw, db if ctx.has[0] else None, dy if ctx.has[1] else None, None, None, None, None


_linear_act_op.register_autograd(_linear_act_op_backward, setup_context=_linear_act_setup)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
               residual: Optional[torch.Tensor] = None, *, algo: str = "dense", depth: int = 0,
               precision: Optional[str] = None) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual as one call, on the current CUDA stream.

    x: (..., K), weight: (N, K), bias: (N,) or None, residual: (..., N) or None; activation one of ``ACTIVATIONS``.
    All of one type (bias is converted); rows may be strided and of any length (operand rows that are not whole
    16-byte vectors are copied). Everything after the product is fp32 and rounded once. Differentiable once in all
    four; for the backward pass the pre-activation is kept in x's type. ``algo``, ``depth`` and ``precision`` choose
    the products, forward and backward, as in `matmul`. Inside torch.compile the layer always keeps the
    pre-activation and its backward pass computes the gradients of x, weight and bias whether needed or not."""
    _call.require_cuda(x, weight, bias, residual)
    if not torch.compiler.is_compiling():
        _call.refuse_tangents(x, weight, bias, residual)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dtype not in _DTYPE or weight.dtype != x.dtype:
        raise TypeError(f"unsupported operand dtypes {x.dtype}, {weight.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not form x @ weight.T")
    if algo not in _ALGO:
        raise ValueError(f"algo must be one of {sorted(_ALGO)}, got {algo!r}")
    if precision is not None:
        resolve_precision(precision)
    out_shape = x.shape[:-1] + (weight.shape[0],)
    if bias is not None:
        if bias.shape != out_shape[-1:]:
            raise ValueError(f"bias must hold {out_shape[-1]} elements, got shape {tuple(bias.shape)}")
        if bias.dtype != x.dtype or not bias.is_contiguous():
            bias = bias.to(x.dtype).contiguous()
    if residual is not None:
        if residual.shape != out_shape:
            raise ValueError(f"residual must have the shape of the result {tuple(out_shape)}, got {tuple(residual.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"residual must be of the type of x ({x.dtype}), got {residual.dtype}")
        if residual.dim() != 2:
            residual = residual.reshape(-1, out_shape[-1])
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    depth = int(depth)
    if (x.dtype != torch.float32 and _rows_contiguous(x2) and _rows_contiguous(weight) and not torch.compiler.is_compiling()
            and (algo == "dense" or (algo == "auto" and x2.shape[0] > 0
                                     and _auto_is_dense(x2.shape[0], weight.shape[0], weight.shape[1], _DTYPE[x.dtype])))):
        if _call.wants_grad(x, weight, bias, residual):
            y = _DenseLinearFn.apply(x2, weight, bias, residual, act)
        else:
            y = _dense_forward(x2, weight, bias, residual, act, False)[0]
    elif torch.compiler.is_compiling():
        y = _linear_act_op(x2, weight, bias, residual, act, algo, depth, precision or "")[0]
    elif _call.wants_grad(x, weight, bias, residual):
        y = _LinearActFn.apply(x2, weight, bias, residual, act, algo, depth, precision)
    else:
        y = _linear_act_forward(x2, weight, bias, residual, act, algo, depth, precision, False)[0]
    return y if x.dim() == 2 else y.view(out_shape)
