"""The global gradient norm and clipping against the formula in 64 bits.

Tolerances: the sum of squares is fp64, so the norm is off by its rounding to fp32 (2^-24) and a few 2^-50;
a clipped value by the rounding of the coefficient, of the product (2^-24 each) and of the result (eps/2).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b200s(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    import strassen_triton_b200

    return strassen_triton_b200


def norm64(grads):
    return math.sqrt(sum(t.double().square().sum().item() for t in grads))


def check(got, src, coef):
    ref = src.double() * coef
    fi = torch.finfo(got.dtype)
    tol = ref.abs() * (2.0 ** -22 + fi.eps / 2 * 1.01) + fi.smallest_normal * fi.eps
    assert ((got.double() - ref).abs() <= tol).all()


def make(sizes, dtypes, seed=0, scale=1e-2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


ALL = [torch.bfloat16, torch.float32, torch.float16]
LISTS = [[1], [0, 5], [7, 8, 9, 31, 32, 33], [16384, 16385, 16383, 1], [100000], [3] * 400, [5_000_003, 17, 1_000_000], list(range(1, 300, 7))]


@pytest.mark.parametrize("sizes", LISTS, ids=[str(len(s)) + "x" + str(max(s)) for s in LISTS])
@pytest.mark.parametrize("dtypes", [[torch.bfloat16], [torch.float32], ALL], ids=["bf16", "fp32", "mixed"])
def test_norm_and_clipping(b200s, sizes, dtypes):
    grads = make(sizes, dtypes)
    want = norm64(grads)
    got = b200s.grad_norm(grads)
    assert got.dtype == torch.float32 and got.shape == () and abs(got.item() - want) <= 2.0 ** -23 * want
    for bound in (want * 0.37, want * 3):
        coef = min(1.0, bound / (want + 1e-6))
        mine = [t.clone() for t in grads]
        n = b200s.clip_grads_(mine, bound)
        assert torch.equal(n, got)
        for a, t in zip(mine, grads):
            check(a, t, coef)
            if coef == 1.0:
                assert torch.equal(a, t)
        for odt in ALL:
            out = [torch.full_like(t, float("nan"), dtype=odt) for t in grads]
            keep = [t.clone() for t in grads]
            b200s.clip_grads_(keep, bound, out=out)
            assert all(torch.equal(a, b) for a, b in zip(keep, grads))
            for a, t in zip(out, grads):
                check(a, t, coef)


@pytest.mark.parametrize("dtype", ALL)
def test_views_off_alignment_leave_their_neighbours(b200s, dtype):
    """Views at every offset of a flat buffer; what lies between them stays as it was."""
    flat = torch.full((5000,), 3.0, device="cuda", dtype=dtype)
    spans, at = [], 1
    for n in (1, 2, 3, 17, 64, 65, 700, 1000, 31):
        spans.append((at, n))
        at += n + 1
    vals = make([n for _, n in spans], [dtype], scale=1.0)
    for (a, n), v in zip(spans, vals):
        flat[a:a + n] = v
    views = [flat[a:a + n] for a, n in spans]
    out_flat = torch.full((6000,), 5.0, device="cuda")
    outs = [out_flat[a + 2:a + 2 + n] for a, n in spans]
    b200s.clip_grads_(views, 1.0, out=outs)
    b200s.clip_grads_(views, 1.0)
    coef = 1.0 / (norm64(vals) + 1e-6)
    used, used_out = torch.zeros(5000, dtype=torch.bool, device="cuda"), torch.zeros(6000, dtype=torch.bool, device="cuda")
    for (a, n), v, o in zip(spans, vals, outs):
        check(flat[a:a + n], v, coef)
        check(o, v, coef)
        used[a:a + n] = True
        used_out[a + 2:a + 2 + n] = True
    assert (flat[~used] == 3).all() and (out_flat[~used_out] == 5).all()


def test_layouts(b200s):
    """Transposed gradients are taken as they lie; gaps between elements are neither counted nor touched."""
    base = torch.randn(40, 30, device="cuda")
    wide = torch.randn(40, 33, device="cuda")
    keep_base, keep_wide = base.clone(), wide.clone()
    grads = [base.t(), wide[:, 2:31]]
    want = norm64(grads)
    n = b200s.clip_grads_(grads, 1.0)
    assert abs(n.item() - want) <= 2.0 ** -23 * want
    check(base, keep_base, 1 / (want + 1e-6))
    check(wide[:, 2:31], keep_wide[:, 2:31], 1 / (want + 1e-6))
    assert torch.equal(wide[:, :2], keep_wide[:, :2]) and torch.equal(wide[:, 31:], keep_wide[:, 31:])
    out = [torch.empty(30, 40, device="cuda"), torch.empty(29, 40, device="cuda").t()]
    src = [keep_base.t(), keep_wide[:, 2:31]]
    b200s.clip_grads_(src, 1.0, out=out)
    for o, s in zip(out, src):
        check(o, s, 1 / (want + 1e-6))


def test_more_tensors_than_one_launch_takes(b200s):
    grads = make([5 + i % 7 for i in range(1300)], ALL)
    want = norm64(grads)
    out = [torch.empty_like(t, dtype=torch.float32) for t in grads]
    n = b200s.clip_grads_(grads, want / 3, out=out)
    assert abs(n.item() / want - 1) < 2.0 ** -22 and torch.equal(n, b200s.grad_norm(grads))
    for o, t in zip(out, grads):
        check(o, t, (want / 3) / (want + 1e-6))


def test_shards_of_several_ranks(b200s, monkeypatch):
    """With a process group the sums of squares of all ranks are added before the root: here a second rank that holds
    three times the squares."""
    import torch.distributed as dist

    seen = []

    def all_reduce(t, group=None):
        seen.append(group)
        t.mul_(4.0)

    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    grads = make([100, 33], [torch.float32])
    want = 2 * norm64(grads)
    keep = [t.clone() for t in grads]
    assert abs(b200s.grad_norm(grads, group="shards").item() / want - 1) < 2.0 ** -22
    n = b200s.clip_grads_(grads, want / 2, group="shards")
    assert abs(n.item() / want - 1) < 2.0 ** -22 and seen == ["shards", "shards"]
    for a, t in zip(grads, keep):
        check(a, t, (want / 2) / (want + 1e-6))


def test_extreme_and_nonfinite_values(b200s):
    """Squares are fp64: neither 1e30 nor 1e-30 is lost. inf makes the coefficient zero, NaN makes everything NaN."""
    for scale in (1e30, 1e-30):
        g = make([1000, 77], [torch.float32, torch.bfloat16], scale=scale)
        assert abs(b200s.grad_norm(g).item() / norm64(g) - 1) < 2.0 ** -22
    g = make([100, 50], [torch.float32])
    g[1][3] = float("inf")
    assert math.isinf(b200s.clip_grads_(g, 1.0).item())
    assert not g[0].any() and torch.isnan(g[1][3]) and not g[1][:3].any()
    g = make([100, 50], [torch.float32])
    g[0][3] = float("nan")
    keep = [t.clone() for t in g]
    with pytest.raises(RuntimeError):
        b200s.clip_grads_(g, 1.0, error_if_nonfinite=True)
    assert torch.equal(g[1], keep[1])
    assert math.isnan(b200s.clip_grads_(g, 1.0).item()) and torch.isnan(g[0]).all() and torch.isnan(g[1]).all()
    z = [torch.zeros(10, device="cuda")]
    assert b200s.clip_grads_(z, 1.0).item() == 0 and not z[0].any()
    g = make([100], [torch.float32])
    b200s.clip_grads_(g, 0.0)
    assert not g[0].any()
    g = make([100], [torch.float32])
    keep = g[0].clone()
    b200s.clip_grads_(g, float("inf"))
    assert torch.equal(g[0], keep)


def test_parameters_as_torch_does(b200s):
    torch.manual_seed(0)
    a = torch.nn.Sequential(torch.nn.Linear(50, 60), torch.nn.Linear(60, 7)).cuda()
    b = torch.nn.Sequential(torch.nn.Linear(50, 60), torch.nn.Linear(60, 7)).cuda()
    b.load_state_dict(a.state_dict())
    x = torch.randn(20, 50, device="cuda")
    for m in (a, b):
        m(x).square().sum().backward()
    b[1].bias.grad = a[1].bias.grad = None
    na = b200s.clip_grad_norm_(a.parameters(), 0.5)
    nb = torch.nn.utils.clip_grad_norm_(b.parameters(), 0.5)
    assert torch.allclose(na, nb, rtol=1e-5)
    for p, q in zip(a.parameters(), b.parameters()):
        if q.grad is not None:
            assert torch.allclose(p.grad, q.grad, rtol=1e-5, atol=1e-8)
    assert a[1].bias.grad is None


def test_autograd_notices_the_clipping(b200s):
    """A gradient that a second backward pass needs may not be scaled under it silently."""
    x = torch.ones(10, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    loss = (g ** 2).sum()
    b200s.clip_grads_([g.detach()], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals(b200s):
    g = make([10, 20], [torch.float32])
    with pytest.raises(ValueError):
        b200s.clip_grads_([g[0], g[0]], 1.0)                        # the same tensor twice, in place
    with pytest.raises(ValueError):
        b200s.clip_grads_([g[1][:12], g[1][10:]], 1.0)              # overlapping views
    with pytest.raises(ValueError):
        b200s.clip_grads_([g[0].expand(5, 10)], 1.0)
    with pytest.raises(ValueError):
        b200s.clip_grads_(g, -1.0)
    with pytest.raises(ValueError):
        b200s.clip_grads_(g, 1.0, out=[g[1], g[0]])
    with pytest.raises(ValueError):
        b200s.clip_grads_(g, 1.0, out=[g[0].clone()])
    with pytest.raises(TypeError):
        b200s.clip_grads_([g[0].double()], 1.0)
    with pytest.raises(ValueError):
        b200s.grad_norm([])
    with pytest.raises(ValueError):
        b200s.clip_grad_norm_(torch.nn.Parameter(g[0]), 1.0, norm_type=1.0)
    assert abs(b200s.grad_norm([g[0], g[0]]).item() - norm64([g[0], g[0]])) < 1e-6    # reading twice is fine
    assert b200s.clip_grad_norm_([torch.nn.Parameter(g[0])], 1.0).item() == 0


def test_graph_and_repeats(b200s):
    grads = make([1000, 16384 * 3 + 5, 9], ALL)
    out = [torch.empty_like(t) for t in grads]
    n1 = b200s.clip_grads_(grads, 0.1, out=out)
    first = [t.clone() for t in out]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n2 = b200s.clip_grads_(grads, 0.1, out=out)
    for o in out:
        o.zero_()
    g.replay()
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(out, first))
    for t in grads:
        t.mul_(2)
    g.replay()
    assert abs(n2.item() / norm64(grads) - 1) < 2.0 ** -22


def test_tensors_without_memory_are_refused(b200s):
    """A wrapper (a sharded tensor of torch's) has a device and a size, its memory is its local part's."""

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} on a wrapper")

    real = make([100], [torch.float32])[0]
    for grads in ([Wrapper(real)], [real, Wrapper(real)]):
        with pytest.raises(TypeError, match="Wrapper"):
            b200s.grad_norm(grads)
        with pytest.raises(TypeError, match="Wrapper"):
            b200s.clip_grads_(grads, 1.0)


def test_an_empty_list_with_a_group(b200s, monkeypatch):
    import torch.distributed as dist

    monkeypatch.setattr(dist, "all_reduce", lambda t, group=None: t.add_(16.0))
    assert b200s.grad_norm([], group="shards").item() == 4.0
    assert b200s.clip_grads_([], 1.0, group="shards").item() == 4.0
    with pytest.raises(ValueError):
        b200s.grad_norm([])
