"""Gradients of token log probabilities whose logits share a large offset: softmax does not see it, nor may they.

Tolerance, relative to p = e^(x-m) / s (U = 2^-24, g = x - m): g is rounded once, its product with log2 e carries the
constant's rounding and its own (3 U |g| together), the exponential 4 U, log s (c + 16) U + 2 U |log s| with the
chain of c = V / 256 + 40 additions, e^(-log s) 4 U, the products 4 U. Nothing depends on the size of m. The
entropy's gradient adds the errors of log p + H = g + (H - log s). Results are rounded once.
"""
import ctypes

import pytest
import torch

from tests.test_gpu_logprobs import INF, U, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b200s(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    import strassen_triton_b200

    return strassen_triton_b200


def gradient(logits, targets, vocab, dlp, dent):
    """dlogits in 64 bits and its tolerance before the last rounding."""
    x = logits[:, :vocab].double()
    c = vocab / 256 + 40
    gap = x - x.amax(1, keepdim=True)
    s = gap.exp().sum(1, keepdim=True)
    logs = s.log()
    p = gap.exp() / s
    gap = gap.masked_fill(gap == -INF, 0)
    lp = gap - logs
    ent = -(p * lp).sum(1, keepdim=True)
    ignored = targets == -100
    gl = dlp.double().masked_fill(ignored, 0)[:, None]
    ge = dent.double()[:, None]
    t = targets.masked_fill(ignored, 0)[:, None]
    d = -gl * p
    d.scatter_add_(1, t, gl)
    d = d - ge * p * (lp + ent)
    e_log = (c + 16) * U + 2 * U * logs
    e_h = e_log + (c + 48) * U * (p * gap.abs()).sum(1, keepdim=True) + 4 * U
    rel = 3 * U * gap.abs() + e_log + 12 * U
    tol = gl.abs() * p * (rel + 2 * U)
    tol = tol + ge.abs() * p * ((rel + 2 * U) * (lp + ent).abs() + e_h + e_log + 2 * U * (gap.abs() + logs + ent))
    tol.scatter_add_(1, t, 2 * U * gl.abs())
    pad = logits.shape[1] - vocab
    return torch.nn.functional.pad(d, (0, pad)), torch.nn.functional.pad(tol, (0, pad))


@pytest.mark.parametrize("offset", [0.0, 1e3, -1e4, 3e4])
@pytest.mark.parametrize("rows,width,vocab", [(3, 97, 97), (64, 5000, 5000), (5, 50304, 50257), (700, 1001, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_common_offset_does_not_reach_the_gradient(b200s, offset, rows, width, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn(rows, width, generator=g, device="cuda") * 3 + offset).to(dtype)
    x[:, ::7] = -INF                                  # forbidden tokens
    t = torch.randint(0, vocab // 7, (rows,), generator=g, device="cuda") * 7 + 1
    t[::5] = -100
    dlp, dent = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    x.requires_grad_(True)
    r = b200s.token_logprobs(x, t, vocab=vocab, entropy=True)
    d, = torch.autograd.grad((r.logprob, r.entropy), x, (dlp, dent))
    check("dlogits", d, gradient(x.detach(), t, vocab, dlp, dent), dtype)
    d, = torch.autograd.grad(b200s.token_logprobs(x, t, vocab=vocab).logprob, x, dlp)
    check("dlogits of logprob", d, gradient(x.detach(), t, vocab, dlp, torch.zeros_like(dent)), dtype)


def test_both_pairs_of_entries(b200s):
    """The C entries with lse and those with its two parts: the same forward results, lse the sum of the parts, and
    near zero, where lse loses nothing, the same gradients up to the roundings both are allowed."""
    from strassen_triton_b200 import _lib

    lib = _lib.load()
    rows, v = 9, 3001
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, v, generator=g, device="cuda") * 3
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    dlp, dent = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    lp, lp2, lse, ent, ent2 = (torch.empty(rows, device="cuda") for _ in range(5))
    st = torch.empty(rows, 2, device="cuda")
    d, d2 = torch.empty_like(x), torch.empty_like(x)
    s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda a: a.data_ptr()  # noqa: E731
    assert lib.b200s_token_logprobs(rows, v, _lib.FP32, p(x), v, p(t), -100, p(lp), p(lse), p(ent), 0, None, None, s) == 0
    assert lib.b200s_token_logprobs_stats(rows, v, _lib.FP32, p(x), v, p(t), -100, p(lp2), p(st), p(ent2), 0, None, None, s) == 0
    assert torch.equal(lp, lp2) and torch.equal(ent, ent2) and torch.equal(lse, st[:, 0] + st[:, 1])
    assert torch.equal(st[:, 0], x.amax(1))
    args = (rows, v, v, _lib.FP32, p(x), v, p(t), -100)
    assert lib.b200s_token_logprobs_backward(*args, p(lse), p(ent), p(dlp), p(dent), p(d), v, s) == 0
    assert lib.b200s_token_logprobs_backward_stats(*args, p(st), p(ent), p(dlp), p(dent), p(d2), v, s) == 0
    ref, tol = gradient(x, t, v, dlp, dent)
    check("dlogits from the parts", d2, (ref, tol), torch.float32)
    # lse, below 16 here, is rounded by up to 8 U, which goes into every exponent and into log p + H, and the
    # exponents are x - lse instead of x - m, longer by log s < 16: 3 U of that
    y = x.double().log_softmax(1)
    q, ent = y.exp(), -(y.exp() * y).sum(1, keepdim=True)
    assert lse.abs().max() < 16 and st[:, 1].max() < 16
    worst = 64 * U * q * (dlp.double().abs()[:, None] + dent.double().abs()[:, None] * (1 + (y + ent).abs()))
    check("dlogits from lse", d, (ref, tol + worst), torch.float32)
