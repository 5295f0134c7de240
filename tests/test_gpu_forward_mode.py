"""Dual tensors are refused by every differentiable call: none has a forward-mode derivative."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused(built_library):
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    import strassen_triton_b200 as b200s
    from strassen_triton_b200.linear import LinearStrassen

    x, w = torch.randn(32, 64, device="cuda", dtype=torch.bfloat16), torch.randn(16, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(32, dtype=torch.int64, device="cuda")
    plain, act = (LinearStrassen(64, 16, dtype=torch.bfloat16, activation=a) for a in ("none", "gelu"))
    calls = (b200s.layer_norm, lambda x: b200s.linear_act(x, w), lambda x: b200s.token_logprobs(x, t),
             lambda x: b200s.cross_entropy(x, t), lambda x: b200s.matmul_autograd(x, w.t()), plain, act,
             lambda x: b200s.linear_act(x.float(), w.float()))
    with forward_ad.dual_level():
        for call in calls:
            call(x)
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
