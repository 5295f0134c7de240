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
