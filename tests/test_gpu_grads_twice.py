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


def test_an_empty_parameter_list_with_a_group(built_library, monkeypatch):
    """The rank adds nothing to the sum, takes part in it and learns the norm (a stand-in adds the others' squares)."""
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    import torch.distributed as dist

    import strassen_triton_b200 as b200s

    seen = []

    def all_reduce(t, group=None):
        seen.append((group, t.dtype, t.tolist(), t.is_cuda))
        t.add_(25.0)

    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    n = b200s.clip_grad_norm_([], 1.0, group="stages")
    assert n.is_cuda and n.shape == () and n.dtype == torch.float32 and n.item() == 5.0
    assert seen == [("stages", torch.float64, [0.0], True)]
