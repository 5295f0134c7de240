"""Rows of one value: nothing is left of them but the bias."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [1, 3, 7, 100, 768, 1000, 1601, 2050, 4096, 5000, 8190, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [3, 600])
def test_rows_of_one_value_give_the_bias(built_library, d, dtype, rows):
    """Values of 11 bits in rows of up to 8192, of 8 bits in longer ones: every sum of them fits the 24 bits of fp32, so
    the mean is the value itself, x - mean is 0 and the result the bias, exactly; with a mean that is a rounding off
    it is noise of up to 0.8."""
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    import strassen_triton_b200 as b200s

    values = torch.tensor([1000.0, -12345.678, 0.1, 54321.0, 3.0, 60000.0], device="cuda").to(torch.float16)
    values = (values.to(torch.bfloat16) if d > 8192 else values).to(dtype)
    x = values[torch.arange(rows, device="cuda") % len(values)][:, None].repeat(1, d)
    b = torch.linspace(-1, 1, d, device="cuda").to(dtype)
    w = torch.full_like(b, 1.5)
    assert torch.equal(b200s.layer_norm(x, w, b), b.expand(rows, d))
    x.requires_grad_(True)
    y = b200s.layer_norm(x, w, b)
    assert torch.equal(y.detach(), b.expand(rows, d))
    # xhat is 0: dx = rstd (g - mean(g)), zero for a gradient that is the same everywhere up to the mean's rounding
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx.abs().max() <= 1e-5 ** -0.5 * 1.5 * (d / 32 + 42) * 2.0 ** -24
