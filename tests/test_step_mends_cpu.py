"""Calls of the training-step operators that lost something in silence, on a machine without a GPU."""
import pytest
import torch


def test_a_rank_without_parameters_takes_part_in_the_norm(monkeypatch):
    """A pipeline stage without trainable parameters: the other ranks wait in their all-reduce for it."""
    from strassen_triton_b200 import grads

    calls = []

    def no_share(device, group, error_if_nonfinite=False):
        calls.append((group, error_if_nonfinite))
        return torch.tensor(3.0)

    monkeypatch.setattr(grads, "_no_share", no_share)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    assert grads.clip_grad_norm_([], 1.0, group="shards").item() == 3.0
    assert grads.clip_grad_norm_(iter(()), 1.0, error_if_nonfinite=True, group="shards").item() == 3.0
    assert calls == [("shards", False), ("shards", True)]
    with pytest.raises(ValueError):
        grads.clip_grad_norm_([], -1.0, group="shards")
    assert grads.clip_grad_norm_([], 1.0).item() == 0.0 and len(calls) == 2      # without a group nobody waits


def test_logprob_entries_with_statistics_in_two_parts(built_library):
    from strassen_triton_b200 import _lib

    lib = _lib.load()
    args = dict(rows=4, vocab=8, dt=_lib.BF16, x=16, ld=8, t=16, ig=-100, lp=16, st=16, ent=16, k=2, ids=16, top=16)
    call = lambda **kw: lib.b200s_token_logprobs_stats(*{**args, **kw}.values(), None)  # noqa: E731
    assert call(st=20) == _lib.ERR_BAD_ALIGNMENT and call(k=9) == _lib.ERR_BAD_SHAPE and call(t=None) == _lib.ERR_NULL_POINTER
    assert call(rows=0, x=None) == 0
    args = dict(rows=4, vocab=8, width=8, dt=_lib.BF16, x=16, ld=8, t=16, ig=-100, st=16, ent=16, dl=16, de=16, out=16, ldd=8)
    back = lambda **kw: lib.b200s_token_logprobs_backward_stats(*{**args, **kw}.values(), None)  # noqa: E731
    assert back(st=20) == _lib.ERR_BAD_ALIGNMENT and back(st=None) == _lib.ERR_NULL_POINTER and back(ent=None) == _lib.ERR_NULL_POINTER


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """The operators have none: a dual tensor must not come out without its tangent (the kernels are stand-ins here)."""
    import torch.autograd.forward_ad as forward_ad

    from strassen_triton_b200 import _call, loss, norm, ops

    for module in (loss, norm, ops):
        if hasattr(module, "require_cuda"):
            monkeypatch.setattr(module, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_call, "require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: None)
    ran = []
    monkeypatch.setattr(norm, "_forward", lambda x, *a: (ran.append("norm"), x))
    monkeypatch.setattr(loss, "_forward", lambda x, *a: ran.append("loss") or (x[..., 0], None, None, None, None))
    monkeypatch.setattr(ops, "_dense_forward", lambda x, w, *a: ran.append("linear") or (x @ w.t(), None))
    monkeypatch.setattr(ops, "_linear_act_forward", lambda x, w, *a: ran.append("linear") or (x @ w.t(), None))
    monkeypatch.setattr(ops, "_matmul_op", lambda x, w, *a: ran.append("matmul") or x @ w)
    monkeypatch.setattr(ops, "_linear_op", lambda x, w, b, *a: ran.append("matmul") or x @ w + b)
    x, w, b, t = torch.randn(4, 8), torch.randn(8, 8), torch.randn(8), torch.zeros(4, dtype=torch.int64)
    calls = (lambda x, w, b: norm.layer_norm(x, b, b), lambda x, w, b: ops.linear_act(x, w, b),
             lambda x, w, b: ops.linear_act(x.bfloat16(), w.bfloat16(), b), lambda x, w, b: loss.token_logprobs(x, t),
             lambda x, w, b: loss.cross_entropy(x, t), lambda x, w, b: ops.matmul_autograd(x, w),
             lambda x, w, b: ops.linear_autograd(x, w, b))
    for call in calls:
        call(x, w, b)
    n = len(ran)
    with forward_ad.dual_level():
        dual = lambda v: forward_ad.make_dual(v, torch.ones_like(v))  # noqa: E731
        for k, call in enumerate(calls):
            call(x, w, b)                     # plain tensors at a dual level are fine
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual(x), w, b)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual(x), w, b)
            if k not in (3, 4):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(x, w, dual(b)) if k in (0, 1, 2, 6) else call(x, dual(w), b)
    assert len(ran) == 2 * n
