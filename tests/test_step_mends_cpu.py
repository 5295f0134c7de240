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
