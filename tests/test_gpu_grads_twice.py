"""A gradient that is written may not be in the list twice, whatever its layout."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_strided_tensor_given_twice_is_refused(built_library):
    """Rows of a wider matrix are scaled through a copy, so the list the kernels see has no overlap."""
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    import strassen_triton_b200 as b200s

    wide = torch.ones(8, 12, device="cuda")
    view, other = wide[:, 1:5], wide[:, 6:10]
    with pytest.raises(ValueError, match="twice"):
        b200s.clip_grads_([view, other, view], 0.1)
    out = torch.zeros(8, 12, device="cuda")[:, :4]
    with pytest.raises(ValueError, match="twice"):
        b200s.clip_grads_([torch.ones(8, 4, device="cuda"), torch.ones(8, 4, device="cuda")], 0.1, out=[out, out])
    assert (wide == 1).all() and not out.any()            # refused before anything was written
    # what is only read may repeat (four times 32 ones; sqrt(128) is rounded once)
    assert abs(b200s.grad_norm([view, view, other, other]).item() - 128.0 ** 0.5) <= 128.0 ** 0.5 * 2.0 ** -24
    empty = wide[:, 1:5][:0]
    assert b200s.clip_grads_([empty, empty, view, other], 0.1).item() == 8.0
    assert torch.allclose(view, torch.full_like(view, 0.1 / 8), rtol=1e-5)
