"""Refusals of the training-step operators on a machine without a GPU: the C entries look at their arguments
before any device, the tensor-level calls have no CPU path."""
import ctypes

import pytest
import torch

from strassen_triton_b200 import _lib


@pytest.fixture(scope="module")
def lib(built_library):
    return _lib.load()


def test_layer_norm_arguments(lib):
    f = lib.b200s_layer_norm
    ok = dict(rows=4, d=8, dt=_lib.BF16, pd=_lib.BF16, eps=1e-5, x=16, ldx=8, w=16, b=16, y=16, ldy=8, m=None, r=None)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None)

    assert call(rows=-1) == _lib.ERR_BAD_SHAPE and call(d=0) == _lib.ERR_BAD_SHAPE
    assert call(dt=5) == _lib.ERR_BAD_DTYPE and call(pd=_lib.FP16) == _lib.ERR_BAD_DTYPE
    assert call(eps=-1.0) == _lib.ERR_BAD_SHAPE and call(eps=float("nan")) == _lib.ERR_BAD_SHAPE
    assert call(x=None) == _lib.ERR_NULL_POINTER and call(y=None) == _lib.ERR_NULL_POINTER
    assert call(m=16) == _lib.ERR_NULL_POINTER
    assert call(ldy=7) == _lib.ERR_BAD_STRIDE and call(ldx=-8) == _lib.ERR_BAD_STRIDE
    assert call(x=17) == _lib.ERR_BAD_ALIGNMENT and call(w=17) == _lib.ERR_BAD_ALIGNMENT
    assert call(rows=0, x=None, y=None) == 0
    n = ctypes.c_size_t(0)
    assert lib.b200s_layer_norm_backward_workspace(4, 8, None) == _lib.ERR_NULL_POINTER
    assert lib.b200s_layer_norm_backward_workspace(4, 8, ctypes.byref(n)) == 0 and n.value >= 2 * 8 * 4
    g = lib.b200s_layer_norm_backward
    args = dict(rows=4, d=8, dt=_lib.BF16, pd=_lib.BF16, x=16, ldx=8, dy=16, ldg=8, w=16, m=16, r=16, dx=16, lddx=8, dw=16,
                db=16, ws=16, n=1 << 20)

    def back(**kw):
        return g(*{**args, **kw}.values(), None)

    assert back(n=4) == _lib.ERR_WORKSPACE_TOO_SMALL and back(ws=None) == _lib.ERR_NULL_POINTER
    assert back(ws=24) == _lib.ERR_BAD_ALIGNMENT and back(dy=None) == _lib.ERR_NULL_POINTER
    assert back(lddx=7) == _lib.ERR_BAD_STRIDE and back(dy=17) == _lib.ERR_BAD_ALIGNMENT


def problem(**kw):
    p = _lib.Problem()
    p.M, p.N, p.K, p.batch = 64, 48, 32, 1
    p.lda, p.ldb, p.ldc = 32, 32, 48
    p.a_major, p.b_major = _lib.K_MAJOR, _lib.K_MAJOR
    p.algo, p.prod_dtype = _lib.ALGO_DENSE, -1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_epilogue_arguments(lib):
    n = ctypes.c_size_t(0)
    e = _lib.Epilogue()
    ws = lambda p, e: lib.b200s_matmul_epilogue_workspace(ctypes.byref(p), ctypes.byref(e), ctypes.byref(n))  # noqa: E731
    assert ws(problem(), e) == 0
    assert ws(problem(beta=1), e) == _lib.ERR_BAD_SHAPE and ws(problem(batch=2), e) == _lib.ERR_BAD_SHAPE
    assert ws(problem(ldc=40), e) == _lib.ERR_BAD_STRIDE and ws(problem(M=0), e) == _lib.ERR_BAD_SHAPE
    assert ws(problem(out_dtype=9), e) == _lib.ERR_BAD_DTYPE
    e.activation = 6
    assert ws(problem(), e) == _lib.ERR_BAD_ALGO
    e.activation, e.residual, e.ld_residual = _lib.ACT_GELU, 16, -1
    assert ws(problem(), e) == _lib.ERR_BAD_STRIDE
    e.ld_residual, e.preact, e.ld_preact = 48, 16, 40
    assert ws(problem(), e) == _lib.ERR_BAD_STRIDE
    e.ld_preact, e.bias = 48, 17
    assert ws(problem(), e) == _lib.ERR_BAD_ALIGNMENT
    e.bias = 16
    run = lambda A, B, C, w, k: lib.b200s_matmul_epilogue(ctypes.byref(problem()), ctypes.byref(e), A, B, C, w, k, None)  # noqa: E731
    assert run(None, 16, 16, 256, 1 << 30) == _lib.ERR_NULL_POINTER and run(16, 16, None, 256, 1 << 30) == _lib.ERR_NULL_POINTER
    assert run(16, 16, 17, 256, 1 << 30) == _lib.ERR_BAD_ALIGNMENT
    b = lib.b200s_epilogue_backward
    args = dict(M=4, N=8, dt=_lib.BF16, act=_lib.ACT_GELU, z=16, ldz=8, dy=16, ldy=8, dz=16, lddz=8, db=16, ws=16, n=1 << 20)

    def back(**kw):
        return b(*{**args, **kw}.values(), None)

    assert back(act=-1) == _lib.ERR_BAD_ALGO and back(z=None) == _lib.ERR_NULL_POINTER and back(lddz=7) == _lib.ERR_BAD_STRIDE
    assert back(dz=None, db=None) == _lib.ERR_NULL_POINTER and back(n=0) == _lib.ERR_WORKSPACE_TOO_SMALL
    assert back(N=0) == _lib.ERR_BAD_SHAPE and back(dt=3) == _lib.ERR_BAD_DTYPE and back(dy=17) == _lib.ERR_BAD_ALIGNMENT


def test_linear_arguments(lib):
    n = ctypes.c_size_t(0)
    size = ctypes.byref(n)
    assert lib.b200s_linear_act_workspace(4, 8, 8, _lib.FP32, 0, size) == _lib.ERR_BAD_DTYPE
    assert lib.b200s_linear_act_workspace(4, 0, 8, _lib.BF16, 0, size) == _lib.ERR_BAD_SHAPE
    assert lib.b200s_linear_act_workspace(4, 8, 8, _lib.BF16, 0, None) == _lib.ERR_NULL_POINTER
    assert lib.b200s_linear_act_workspace(4, 8, 8, _lib.BF16, 0, size) == 0 and n.value == 0
    assert lib.b200s_linear_act_workspace(4, 8, 7, _lib.BF16, 1, size) == 0 and n.value >= (4 + 8) * 8 * 2
    f = lib.b200s_linear_act
    args = dict(M=4, N=8, K=8, dt=_lib.BF16, act=_lib.ACT_GELU, x=16, ldx=8, w=16, ldw=8, b=16, r=16, ldr=8, y=16, ldy=8, z=16,
                ldz=8, ws=None, n=0)

    def call(**kw):
        return f(*{**args, **kw}.values(), None)

    assert call(x=None) == _lib.ERR_NULL_POINTER and call(act=7) == _lib.ERR_BAD_ALGO and call(ldy=7) == _lib.ERR_BAD_STRIDE
    assert call(ldz=7) == _lib.ERR_BAD_STRIDE and call(ldx=-8) == _lib.ERR_BAD_STRIDE and call(r=17) == _lib.ERR_BAD_ALIGNMENT
    assert call(x=18) == _lib.ERR_NULL_POINTER                     # a copy of x needs scratch
    assert call(x=18, ws=256, n=16) == _lib.ERR_WORKSPACE_TOO_SMALL and call(x=18, ws=128, n=1 << 20) == _lib.ERR_BAD_ALIGNMENT
    assert call(M=0, x=None, y=None) == 0
    g = lib.b200s_linear_act_backward
    args2 = dict(M=4, N=8, K=8, dt=_lib.BF16, act=_lib.ACT_GELU, x=16, ldx=8, w=16, ldw=8, z=16, ldz=8, dy=16, ldy=8, dx=16, lddx=8,
                 dw=16, lddw=8, db=16, ws=256, n=1 << 20)

    def back(**kw):
        return g(*{**args2, **kw}.values(), None)

    assert back(z=None) == _lib.ERR_NULL_POINTER and back(dy=None) == _lib.ERR_NULL_POINTER and back(ws=None) == _lib.ERR_NULL_POINTER
    assert back(n=8) == _lib.ERR_WORKSPACE_TOO_SMALL and back(lddx=7) == _lib.ERR_BAD_STRIDE and back(dw=17) == _lib.ERR_BAD_ALIGNMENT
    assert back(dx=None, dw=None, db=None) == 0


def test_linear_extents(lib):
    """The far end of the last tile must have 32-bit coordinates: extents within 65536 of 2^31 are refused by both
    ways to the kernels, before any of them runs."""
    n = ctypes.c_size_t(0)
    top = 2 ** 31 - 1 - 65536
    for M, N, K in ((top + 1, 8, 8), (4, top + 1, 8), (4, 8, top + 1), (2 ** 31 - 1, 8, 8)):
        assert lib.b200s_linear_act_workspace(M, N, K, _lib.BF16, 0, ctypes.byref(n)) == _lib.ERR_BAD_SHAPE
        assert lib.b200s_linear_act_backward_workspace(M, N, K, _lib.BF16, _lib.ACT_NONE, 0, ctypes.byref(n)) == _lib.ERR_BAD_SHAPE
        assert lib.b200s_linear_act(M, N, K, _lib.BF16, 0, 16, K, 16, K, None, None, 0, 16, N, None, 0, None, 0, None) == _lib.ERR_BAD_SHAPE
    assert lib.b200s_linear_act_workspace(4, top, 8, _lib.BF16, 0, ctypes.byref(n)) == 0


def test_logprob_arguments(lib):
    f = lib.b200s_token_logprobs
    args = dict(rows=4, vocab=8, dt=_lib.BF16, x=16, ld=8, t=16, ig=-100, lp=16, lse=16, ent=16, k=2, ids=16, top=16)

    def call(**kw):
        return f(*{**args, **kw}.values(), None)

    assert call(vocab=0) == _lib.ERR_BAD_SHAPE and call(k=9) == _lib.ERR_BAD_SHAPE and call(k=-1) == _lib.ERR_BAD_SHAPE
    assert call(vocab=1000, ld=1000, k=65) == _lib.ERR_BAD_SHAPE and call(dt=4) == _lib.ERR_BAD_DTYPE
    assert call(t=None) == _lib.ERR_NULL_POINTER and call(ids=None) == _lib.ERR_NULL_POINTER and call(ld=-8) == _lib.ERR_BAD_STRIDE
    assert call(x=17) == _lib.ERR_BAD_ALIGNMENT and call(t=20) == _lib.ERR_BAD_ALIGNMENT
    assert call(rows=0, x=None) == 0
    g = lib.b200s_token_logprobs_backward
    args2 = dict(rows=4, vocab=8, width=8, dt=_lib.BF16, x=16, ld=8, t=16, ig=-100, lse=16, ent=16, dl=16, de=16, out=16, ldd=8)

    def back(**kw):
        return g(*{**args2, **kw}.values(), None)

    assert back(width=7) == _lib.ERR_BAD_SHAPE and back(ldd=7) == _lib.ERR_BAD_STRIDE and back(ent=None) == _lib.ERR_NULL_POINTER
    assert back(lse=None) == _lib.ERR_NULL_POINTER and back(out=17) == _lib.ERR_BAD_ALIGNMENT


def entries(*spans):
    arr = (_lib.TensorEntry * len(spans))()
    for e, (s, d, n, dt, ddt) in zip(arr, spans):
        e.src, e.dst, e.numel, e.dtype, e.dst_dtype = s, d, n, dt, ddt
    return arr


def test_gradient_list_arguments(lib):
    good = entries((256, 256, 10, 2, 2))
    assert lib.b200s_grad_sumsq(good, -1, 16, None) == _lib.ERR_BAD_SHAPE
    assert lib.b200s_grad_sumsq(None, 1, 16, None) == _lib.ERR_NULL_POINTER
    assert lib.b200s_grad_sumsq(good, 1, None, None) == _lib.ERR_NULL_POINTER
    assert lib.b200s_grad_sumsq(entries((256, 0, 10, 7, 2)), 1, 16, None) == _lib.ERR_BAD_DTYPE
    assert lib.b200s_grad_sumsq(entries((258, 0, 10, 2, 2)), 1, 16, None) == _lib.ERR_BAD_ALIGNMENT
    assert lib.b200s_grad_norm(None, 1, 16, None) == _lib.ERR_NULL_POINTER
    assert lib.b200s_grad_norm(16, _lib.NORM_PARTS + 1, 16, None) == _lib.ERR_BAD_SHAPE
    clip = lambda arr, mx=1.0: lib.b200s_grad_clip(arr, len(arr), 16, 1, mx, 16, None)  # noqa: E731
    assert clip(good, -1.0) == _lib.ERR_BAD_SHAPE and clip(good, float("nan")) == _lib.ERR_BAD_SHAPE
    assert clip(entries((256, 0, 10, 2, 2))) == _lib.ERR_NULL_POINTER
    assert clip(entries((256, 256, 10, 2, 0))) == _lib.ERR_BAD_DTYPE             # in place, but another type
    assert clip(entries((256, 256, 10, 2, 2), (256, 256, 10, 2, 2))) == _lib.ERR_OVERLAP
    assert clip(entries((256, 256, 10, 2, 2), (292, 512, 10, 2, 2))) == _lib.ERR_OVERLAP   # reads what the first writes
    assert clip(entries((256, 1024, 10, 2, 2), (512, 1060, 10, 2, 2))) == _lib.ERR_OVERLAP  # two results overlap
    assert clip(entries((256, 270, 10, 2, 2))) in (_lib.ERR_OVERLAP, _lib.ERR_BAD_ALIGNMENT)


def test_tensor_level_calls_refuse_cpu_tensors_and_bad_arguments():
    import strassen_triton_b200 as b200s

    x, w = torch.ones(2, 8), torch.ones(4, 8)
    for call in (lambda: b200s.layer_norm(x), lambda: b200s.linear_act(x, w),
                 lambda: b200s.token_logprobs(x, torch.zeros(2, dtype=torch.int64)), lambda: b200s.grad_norm([x]),
                 lambda: b200s.clip_grads_([x], 1.0)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        b200s.layer_norm([1.0])
    with pytest.raises(ValueError):
        b200s.cross_entropy(x, torch.zeros(2, dtype=torch.int64), reduction="median")
    with pytest.raises(ValueError):
        b200s.clip_grad_norm_([], 1.0, norm_type=1)


def test_a_rank_without_gradients_takes_part_in_the_norm(monkeypatch):
    """The other ranks wait in their all-reduce for it (a stand-in adds their squares here)."""
    import torch.distributed as dist

    import strassen_triton_b200 as b200s

    calls = []

    def all_reduce(t, group=None):
        calls.append((group, t.dtype, t.tolist()))
        t.add_(float(add))

    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    params = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(2, 2))]
    add = 9.0
    n = b200s.clip_grad_norm_(params, 1.0, group="shards")
    assert n.shape == () and n.dtype == torch.float32 and n.item() == 3.0
    assert calls == [("shards", torch.float64, [0.0])]
    assert b200s.clip_grad_norm_((p for p in params), 1.0).item() == 0.0 and len(calls) == 1
    with pytest.raises(ValueError):
        b200s.clip_grad_norm_(params, -1.0, group="shards")
    assert len(calls) == 1
    add = "nan"
    with pytest.raises(RuntimeError, match="not finite"):
        b200s.clip_grad_norm_(params, 1.0, error_if_nonfinite=True, group="shards")


def test_residual_of_another_shape_is_refused():
    """As many elements in other rows must not be added in silence."""
    from strassen_triton_b200.linear import LinearStrassen

    layer = LinearStrassen(8, 16, device="cpu", depth=0)
    with pytest.raises(ValueError, match="residual"):
        layer(torch.ones(2, 3, 8), residual=torch.ones(3, 2, 16))
    with pytest.raises(ValueError, match="residual"):
        layer(torch.ones(2, 3, 8), residual=torch.ones(6, 16))


def test_dense_layouts():
    from strassen_triton_b200.grads import _dense

    t = torch.empty(4, 5, 6)
    assert _dense(t) and _dense(t.permute(2, 0, 1)) and _dense(t[:1]) and _dense(torch.empty(3, 1).expand(3, 1))
    assert not _dense(t[:, 1:]) and not _dense(t[:, :, ::2]) and not _dense(torch.empty(1, 3).expand(2, 3))
