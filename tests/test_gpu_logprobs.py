"""Token log probabilities, entropies, alternatives and their gradient against the formula in 64 bits.

Tolerances. m is exact. Every term e^(x-m) carries |x-m| 2^-23 + 2^-22 of itself and the sums a chain of
c = V / 256 + 40 additions of positive terms, so log s is good to (c + 16) 2^-24 (the terms far below m weigh
nothing), and logprob = (x_t - m) - log s to that plus 2^-23 of its parts. u / s weighs the same terms with
x - m: (c + 48) 2^-24 of sum e|x-m| / s. p = e^(x - lse) carries (|x - lse| + |lse| + c + 16) 2^-23 of itself. Gradients are
rounded once to the type of the logits.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module")
def b200s(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    import strassen_triton_b200

    return strassen_triton_b200


def reference(logits, targets, vocab, ignore=-100, dlp=None, dent=None):
    x = logits[:, :vocab].double()
    c = vocab / 256 + 40
    m = x.amax(1, keepdim=True)
    empty = (m == -INF)[:, 0]
    m = m.masked_fill(empty[:, None], 0)
    e = (x - m).exp()
    s = e.sum(1, keepdim=True)
    gap = torch.where(e > 0, x - m, torch.zeros_like(x))
    us = (e * gap).sum(1, keepdim=True) / s.masked_fill(empty[:, None], 1)
    lse = m + s.log()
    lp = x - lse
    p = lp.exp()
    ignored = targets == ignore
    t = targets.masked_fill(ignored, 0)[:, None]
    picked = torch.where(empty, torch.full_like(lse[:, 0], -INF), lp.gather(1, t)[:, 0]).masked_fill(ignored, 0)
    e_log = ((c + 16) * U + 2 * U * s.log().abs()[:, 0]).masked_fill(empty, 0)      # nothing is rounded in an empty row
    out = {"logprob": (picked, e_log + 4 * U * torch.nan_to_num(picked, 0, 0, 0).abs())}
    h = (s.log() - us)[:, 0].masked_fill(empty, 0)
    e_h = e_log + (c + 48) * U * us.abs()[:, 0] + 4 * U
    out["entropy"] = (h, e_h)
    if dlp is not None or dent is not None:
        gl = torch.zeros_like(h) if dlp is None else dlp.double().masked_fill(ignored, 0)
        ge = torch.zeros_like(h) if dent is None else dent.double()
        plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        d = -gl[:, None] * p
        d.scatter_add_(1, t, gl[:, None])
        d = d - ge[:, None] * (plp + p * h[:, None])
        d[empty] = 0
        rel = (torch.where(p > 0, lp.abs(), torch.zeros_like(p)) + lse.abs().nan_to_num(0, 0, 0) + c + 16) * 2 * U
        tol = rel * p * gl.abs()[:, None] + ge.abs()[:, None] * (rel * (plp.abs() + p * h[:, None].abs() + p) + p * e_h[:, None])
        tol = tol + 4 * U * gl.abs()[:, None] * (torch.arange(vocab, device=x.device)[None] == t)
        tol[empty] = 0
        pad = logits.shape[1] - vocab
        out["dlogits"] = (torch.nn.functional.pad(d, (0, pad)), torch.nn.functional.pad(tol.nan_to_num(0), (0, pad)))
    return out, lp


def half_step(ref, dtype):
    return ref.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(name, got, want, dtype=torch.float32):
    ref, tol = want
    assert got.dtype == dtype and got.shape == ref.shape
    same_inf = (got.double() == ref) & torch.isinf(ref)
    tol = tol * 1.01 + half_step(ref.abs() + tol, dtype) + 1e-37
    err = torch.where(same_inf, torch.zeros_like(ref), (got.double() - ref).abs())
    worst = (err / torch.where(same_inf, torch.ones_like(tol), tol)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: error is {worst:.2f} of the tolerance"


def check_top(got_ids, got_lp, x, lp, k):
    ids = torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(got_ids, ids)
    want = lp.gather(1, ids)
    want = torch.where(torch.isnan(want), torch.full_like(want, -INF), want)
    c = x.shape[1] / 256 + 40
    check("top_logprobs", got_lp, (want, (c + 16) * U + 4 * U * torch.nan_to_num(want, 0, 0, 0).abs() + 2 * U * lp.isfinite().sum(1, keepdim=True).double().log()))


def make(rows, width, vocab, dtype, masked=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + vocab)
    x = torch.randn(rows, width, generator=g, device="cuda") * 3
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if masked:
        x[torch.rand(rows, width, generator=g, device="cuda") < 0.4] = -INF
        x[rows // 2] = -INF                       # a row with nothing left
    x[:, vocab:] = 1e4 if dtype != torch.float16 else 6e4     # padding must not count
    t[::5] = -100
    dlp = torch.randn(rows, generator=g, device="cuda")
    dent = torch.randn(rows, generator=g, device="cuda") * 0.3
    return x.to(dtype), t, dlp, dent


SHAPES = [(1, 1, 1), (2, 2, 2), (5, 7, 7), (3, 100, 97), (64, 1000, 1000), (7, 4099, 4099), (1, 50304, 50257), (8, 50304, 50257),
          (33, 32003, 32003), (300, 2048, 2000), (4, 131072, 131072), (1, 131073, 131073), (2000, 65, 65)]


@pytest.mark.parametrize("rows,width,vocab", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("masked", [False, True])
def test_everything(b200s, rows, width, vocab, dtype, masked):
    x, t, dlp, dent = make(rows, width, vocab, dtype, masked)
    k = min(vocab, 8)
    want, lp = reference(x, t, vocab, -100, dlp, dent)
    r = b200s.token_logprobs(x, t, vocab=vocab, entropy=True, top_k=k)
    check("logprob", r.logprob, want["logprob"])
    check("entropy", r.entropy, want["entropy"])
    check_top(r.top_ids, r.top_logprobs, x[:, :vocab], lp, k)
    plain = b200s.token_logprobs(x, t, vocab=vocab)
    assert plain.entropy is None and plain.top_ids is None and torch.equal(plain.logprob, r.logprob)
    xg = x.clone().requires_grad_(True)
    r = b200s.token_logprobs(xg, t, vocab=vocab, entropy=True, top_k=k)
    check("logprob", r.logprob.detach(), want["logprob"])
    d, = torch.autograd.grad((r.logprob, r.entropy), xg, (dlp, dent))
    check("dlogits", d, want["dlogits"], dtype)
    xg = x.clone().requires_grad_(True)
    d, = torch.autograd.grad(b200s.token_logprobs(xg, t, vocab=vocab).logprob, xg, dlp)
    check("dlogits of logprob", d, reference(x, t, vocab, -100, dlp)[0]["dlogits"], dtype)
    assert not d[:, vocab:].any() and not d[t == -100].any()


@pytest.mark.parametrize("k", [1, 5, 64])
@pytest.mark.parametrize("kind", ["equal", "few_levels", "ascending", "descending", "one_alive", "signed_zeros"])
def test_alternatives_with_ties(b200s, k, kind):
    """Ties go to the lower id: whole rows of one value, rows of a few values, sorted rows, rows where fewer than k
    tokens are allowed."""
    rows, v = 6, 9001
    g = torch.Generator(device="cuda").manual_seed(5)
    if kind == "equal":
        x = torch.full((rows, v), 1.5, device="cuda")
    elif kind == "few_levels":
        x = torch.randint(0, 3, (rows, v), generator=g, device="cuda").float()
    elif kind == "ascending":
        x = torch.arange(v, device="cuda").float().expand(rows, v) / 100
    elif kind == "descending":
        x = -torch.arange(v, device="cuda").float().expand(rows, v) / 100
    elif kind == "one_alive":
        x = torch.full((rows, v), -INF, device="cuda")
        x[torch.arange(rows), torch.arange(rows) * 1500 + 7] = 2.0
    else:
        x = torch.where(torch.rand(rows, v, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    x = x.to(torch.bfloat16) if kind not in ("ascending", "descending") else x.contiguous()
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    r = b200s.token_logprobs(x, t, top_k=k)
    check_top(r.top_ids, r.top_logprobs, x, reference(x, t, v)[1], k)


def test_nan_infinite_and_lowest_values(b200s):
    x = torch.randn(8, 500, device="cuda")
    t = torch.arange(8, device="cuda")
    x[1, 77] = float("nan")
    x[2, 78] = INF
    x[3] = torch.finfo(torch.float32).min            # a mask of the type's lowest value: all equal, so uniform
    x[4, 100:] = torch.finfo(torch.float32).min
    t[5], t[6], t[7] = 500, -1, -100                 # out of range, out of range, ignored
    x[7, 3] = float("nan")
    xg = x.clone().requires_grad_(True)
    r = b200s.token_logprobs(xg, t, entropy=True)
    d, = torch.autograd.grad(r.logprob.sum(), xg)
    lp = r.logprob.detach()
    assert torch.isnan(lp[[1, 2, 5, 6]]).all() and torch.isnan(r.entropy[[1, 2]]).all()
    assert abs(lp[3].item() + 6.214608) < 1e-5 and abs(r.entropy[3].item() - 6.214608) < 1e-5
    want, _ = reference(x[[0, 4]], t[[0, 4]], 500, dlp=torch.ones(2, device="cuda"))
    check("logprob", lp[[0, 4]], want["logprob"])
    check("entropy", r.entropy.detach()[[0, 4]], reference(x[[0, 4]], t[[0, 4]], 500)[0]["entropy"])
    check("dlogits", d[[0, 4]], want["dlogits"])
    assert torch.isnan(d[[1, 2, 5, 6]]).any(1).all()
    assert lp[7] == 0 and not d[7].any()             # an ignored row hides what its logits hold


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_shapes(b200s, offset, dtype):
    x, t, dlp, dent = make(12, 1000, 1000, dtype)
    wide = torch.full((12, 1013), 77.0, device="cuda", dtype=dtype)
    wide[:, offset:offset + 1000] = x
    view = wide[:, offset:offset + 1000].detach()
    want, lp = reference(x, t, 1000, dlp=dlp, dent=dent)
    for lg, tt, shape in ((view, t, (12,)), (view.reshape(3, 4, 1000), t.view(3, 4), (3, 4)), (view, t.int(), (12,))):
        lg = lg.requires_grad_(True)
        r = b200s.token_logprobs(lg, tt, entropy=True, top_k=4)
        assert r.logprob.shape == shape and r.top_ids.shape == shape + (4,)
        check("logprob", r.logprob.detach().view(12), want["logprob"])
        d, = torch.autograd.grad((r.logprob, r.entropy), lg, (dlp.view(shape), dent.view(shape)))
        check("dlogits", d.view(12, 1000), want["dlogits"], dtype)
    rep = x[:1].expand(12, 1000)
    check("repeated rows", b200s.token_logprobs(rep, t.abs() % 1000).logprob, reference(rep, t.abs() % 1000, 1000)[0]["logprob"])
    tt = t[::1].repeat_interleave(2)[::2]            # strided targets
    check("strided targets", b200s.token_logprobs(x, tt).logprob, want["logprob"])


def test_empty_and_loss(b200s):
    e = torch.empty(0, 100, device="cuda", requires_grad=True)
    r = b200s.token_logprobs(e, torch.empty(0, dtype=torch.int64, device="cuda"), entropy=True, top_k=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    assert torch.autograd.grad(r.logprob.sum(), e)[0].shape == (0, 100)
    x, t, _, _ = make(50, 320, 300, torch.float32)
    for red in ("mean", "sum", "none"):
        a, b = x.clone().requires_grad_(True), x.clone().double().requires_grad_(True)
        la = b200s.cross_entropy(a, t, vocab=300, reduction=red)
        lb = torch.nn.functional.cross_entropy(b[:, :300], t, reduction=red)
        # fp32 sums of 50 losses, each good to 2^-18
        assert torch.allclose(la.double(), lb, rtol=2.0 ** -17, atol=0 if red != "none" else 2.0 ** -17)
        ga, = torch.autograd.grad(la.sum(), a)
        gb, = torch.autograd.grad(lb.sum(), b)
        assert (ga.double() - gb).abs().max() < 2.0 ** -17


def test_gradient_against_differences(b200s):
    x, t, dlp, dent = make(4, 30, 30, torch.float32)
    t = t.clamp_min(0)
    xg = x.clone().requires_grad_(True)
    r = b200s.token_logprobs(xg, t, entropy=True)
    d, = torch.autograd.grad((r.logprob, r.entropy), xg, (dlp, dent))

    def f(v):
        lp = torch.log_softmax(v, 1)
        return (lp.gather(1, t[:, None])[:, 0] * dlp.double() - (lp.exp() * lp).sum(1) * dent.double()).sum()

    h = 1e-6
    for at in (0, 31, 64, 119):
        lo, hi = x.double(), x.double()
        lo.view(-1)[at] -= h
        hi.view(-1)[at] += h
        assert abs(d.view(-1)[at].item() - ((f(hi) - f(lo)) / (2 * h)).item()) < 2.0 ** -17


def test_graph_replay_and_repeats(b200s):
    x, t, dlp, _ = make(40, 2048, 2000, torch.bfloat16)
    xs = x.clone().requires_grad_(True)

    def step():
        r = b200s.token_logprobs(xs, t, vocab=2000, entropy=True, top_k=4)
        return (r.logprob.detach(), r.entropy.detach(), r.top_ids, torch.autograd.grad(r.logprob, xs, dlp)[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = step(), step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x2, t2, _, _ = make(40, 2048, 2000, torch.bfloat16, seed=77)
    with torch.no_grad():
        xs.copy_(x2)
        t.copy_(t2)
    want = step()
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_offsets_past_32_bits(b200s):
    rows, v = (1 << 31) // 50304 + 3, 50304
    x = torch.zeros(rows, v, device="cuda", dtype=torch.bfloat16)
    tail, t_tail, dlp, _ = make(2, v, v, torch.bfloat16)
    x[-2:] = tail
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    t[-2:] = t_tail.clamp_min(0)
    want, lp = reference(tail, t[-2:], v, dlp=dlp)
    x.requires_grad_(True)
    r = b200s.token_logprobs(x, t, top_k=3)
    check("logprob", r.logprob[-2:].detach(), want["logprob"])
    check_top(r.top_ids[-2:], r.top_logprobs[-2:], tail, lp, 3)
    g = torch.zeros(rows, device="cuda")
    g[-2:] = dlp
    d, = torch.autograd.grad(r.logprob, x, g)
    check("dlogits", d[-2:], want["dlogits"], torch.bfloat16)
