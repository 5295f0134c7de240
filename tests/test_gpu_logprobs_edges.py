"""Rows of logits and targets at the edge of what token log probabilities are defined for."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def b200s(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    import strassen_triton_b200

    return strassen_triton_b200


@pytest.mark.parametrize("vocab,rows", [(3, 1), (500, 2), (9001, 4), (9001, 400)])
@pytest.mark.parametrize("others", [-INF, 0.5, INF])
def test_a_nan_makes_the_alternatives_nan(b200s, vocab, rows, others):
    """Whatever the row's other logits are; the NaN itself is the first of them, then the lowest ids of the others."""
    x = torch.full((rows, vocab), others, device="cuda")
    x[:, 1] = NAN
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    r = b200s.token_logprobs(x, t, entropy=True, top_k=2)
    assert torch.isnan(r.logprob).all() and torch.isnan(r.entropy).all() and torch.isnan(r.top_logprobs).all()
    assert torch.equal(r.top_ids, torch.tensor([1, 0], device="cuda").expand(rows, 2))


@pytest.mark.parametrize("vocab,rows", [(3, 2), (500, 4), (9001, 3)])
def test_a_target_out_of_range_makes_the_gradient_nan_in_an_empty_row_too(b200s, vocab, rows):
    """Its log probability is NaN there as in any other row; a forbidden target's row has no gradient."""
    x = torch.full((rows, vocab), -INF, device="cuda", requires_grad=True)
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    t[0] = vocab
    lp = b200s.token_logprobs(x, t).logprob
    assert torch.isnan(lp[0]) and (lp[1:] == -INF).all()
    d, = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert torch.isnan(d[0]).all() and not d[1:].any()


@pytest.mark.parametrize("vocab,rows", [(50, 2), (9001, 3), (2000, 300)])
def test_the_entropy_does_not_see_the_target(b200s, vocab, rows):
    """An entropy alone has the same gradient for every target: in range, ignored or out of range."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda").requires_grad_(True)
    got = []
    for target in (0, -100, -1, vocab):
        t = torch.full((rows,), target, device="cuda")
        r = b200s.token_logprobs(x, t, entropy=True)
        got.append(torch.autograd.grad(r.entropy.sum(), x)[0])
    assert torch.isfinite(got[0]).all() and got[0].any()
    assert all(torch.equal(got[0], d) for d in got[1:])


@pytest.mark.parametrize("rows,vocab,width", [(1, 50257, 50304), (3, 9001, 9001), (400, 1000, 1003)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_in_the_logits_own_memory(b200s, rows, vocab, width, dtype):
    """The C entry may write the gradient over the logits: the same bits as into another buffer, wherever the target
    lies (a row's head, body and tail, and every block that shares it)."""
    from strassen_triton_b200 import _lib

    lib, code = _lib.load(), {torch.bfloat16: _lib.BF16, torch.float32: _lib.FP32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, width, generator=g, device="cuda") * 3).to(dtype)
    dlp, dent = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    lp, ent, st = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda")
    s, p = torch.cuda.current_stream().cuda_stream, lambda a: a.data_ptr()
    for first in (0, 1, 7, 8, 2047, 2048, vocab // 2, vocab - 3):
        t = (torch.arange(rows, device="cuda") + first) % vocab
        assert lib.b200s_token_logprobs_stats(rows, vocab, code, p(x), width, p(t), -100, p(lp), p(st), p(ent), 0, None, None, s) == 0
        out, own = torch.empty_like(x), x.clone()
        for src, dst in ((x, out), (own, own)):
            assert lib.b200s_token_logprobs_backward_stats(rows, vocab, width, code, p(src), width, p(t), -100, p(st), p(ent),
                                                           p(dlp), p(dent), p(dst), width, s) == 0
        assert torch.equal(out, own)
