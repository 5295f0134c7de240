"""The linear layer with bias, activation and residual in its epilogue, forward and backward, against the
formula in 64 bits.

Tolerances, elementwise. A tensor-core product of K terms adds 16 (8 for TF32) of them at a time into an
fp32 accumulator without rounding to nearest: (K / 8 + 16) steps of 2^-23 of sum |a||b|, plus the split of a
long K into parts (a few fp32 additions, inside the 16). Everything after it is fp32: a few 2^-23 of the
terms; an activation is good to 2^-19 of |z| + |act(z)| (two intrinsic exponentials and a division, and an
approximation of Phi with relative error below 2^-17 for 16-bit results). The result is rounded once: eps/2.
The backward pass sees z rounded to x's type, which moves act' by at most max|act''| eps/2 |z|, and rounds
dz once before the products. relu' jumps at zero, where z may be off by its own error: dy is allowed there.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "relu2", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def b200s(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    import strassen_triton_b200

    return strassen_triton_b200


def act64(z, act):
    F = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: F.relu(z), "relu2": lambda: F.relu(z) ** 2, "silu": lambda: F.silu(z),
            "gelu": lambda: F.gelu(z), "gelu_tanh": lambda: F.gelu(z, approximate="tanh")}[act]()


def dact64(z, act):
    z = z.detach().clone().requires_grad_(True)
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


# largest |act'| and |act''| (relu2: per element below)
LIP = {"none": (1, 0), "relu": (1, 0), "relu2": (None, 2), "silu": (1.1, 0.5), "gelu": (1.13, 0.8), "gelu_tanh": (1.13, 0.85)}


def half_step(ref, dtype):
    return ref.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(name, got, ref, tol, dtype):
    tol = tol * 1.01 + half_step(ref.abs() + tol, dtype)
    err = (got.double() - ref).abs()
    assert got.dtype == dtype and got.shape == ref.shape
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: error is {worst:.2f} of the tolerance"


def prod_err(K, a, b):
    return (K / 8 + 16) * 2.0 ** -23 * (a.abs() @ b.abs())


def run_case(b200s, x, w, b, r, act, dy=None, **kw):
    dt = x.dtype
    half = torch.finfo(dt).eps / 2
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    ez = prod_err(x.shape[1], xd, wd.t())
    if b is not None:
        z = z + b.double()
        ez = ez + 2.0 ** -23 * z.abs()
    lip, lip2 = LIP[act]
    lip = 2 * (z.abs() + ez) if lip is None else lip
    y = act64(z, act)
    ey = lip * ez + 2.0 ** -19 * (y.abs() + z.abs() * (2.0 if act != "none" else 0.0) * (2.0 ** 2 if dt != torch.float32 else 1.0))
    if r is not None:
        y = y + r.double()
        ey = ey + 2.0 ** -23 * y.abs()
    check("y without gradients", b200s.linear_act(x, w, b, act, r, **kw), y, ey, dt)
    if dy is None:
        return
    names = {k: t.clone().requires_grad_(True) for k, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    out = b200s.linear_act(names["x"], names["w"], names.get("b"), act, names.get("r"), **kw)
    check("y", out.detach(), y, ey, dt)
    grads = dict(zip(names, torch.autograd.grad(out, list(names.values()), dy)))
    dyd = dy.double()
    da = dact64(z, act)
    dz = dyd * da
    edz = dyd.abs() * (lip2 * (half * z.abs() + ez) + 2.0 ** -19 * (2 + z.abs()) * 2.0 ** 2)
    if act in ("relu", "relu2"):
        edz = edz + dyd.abs() * (z.abs() <= ez + 2.0 ** -23) * (1 if act == "relu" else 2 * ez)
    rounded = edz + half_step(dz.abs() + edz, dt)
    adz = dz.abs() + rounded
    check("dx", grads["x"], dz @ wd, rounded @ wd.abs() + prod_err(w.shape[0], adz, wd), dt)
    check("dw", grads["w"], dz.t() @ xd, rounded.t() @ xd.abs() + prod_err(x.shape[0], adz.t(), xd), dt)
    if b is not None:
        chain = x.shape[0] / 32 + 200
        check("db", grads["b"], dz.sum(0), edz.sum(0) + chain * 2.0 ** -24 * adz.sum(0), dt)
    if r is not None:
        assert torch.equal(grads["r"], dy)


def inputs(m, k, n, dtype, bias=True, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m * 7 + k * 3 + n)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (r(m, k).to(dtype), (r(n, k) * k ** -0.5).to(dtype), (0.2 * r(n)).to(dtype) if bias else None,
            r(m, n).to(dtype) if residual else None, r(m, n).to(dtype))


SHAPES = [(1, 768, 2304), (1, 8, 8), (2, 13, 5), (3, 64, 1), (7, 771, 100), (8, 1024, 768), (16, 520, 1283), (17, 768, 768),
          (33, 256, 264), (64, 4096, 512), (65, 96, 2000), (128, 128, 128), (129, 72, 520), (200, 1000, 333), (511, 768, 2304),
          (1021, 771, 640), (1024, 2304, 768), (300, 8192, 96)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act", ["gelu", "relu2"])
def test_shapes(b200s, m, k, n, act):
    x, w, b, r, dy = inputs(m, k, n, torch.bfloat16)
    run_case(b200s, x, w, b, r, act, dy)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(4, 264, 392), (150, 200, 312)])
def test_activations_and_types(b200s, act, dtype, m, k, n):
    x, w, b, r, dy = inputs(m, k, n, dtype)
    run_case(b200s, x, w, b, r, act, dy)
    run_case(b200s, x, w, None, None, act, dy)
    run_case(b200s, x, w, b, None, act, dy)
    run_case(b200s, x, w, None, r, act)


@pytest.mark.parametrize("m", [1, 8, 16, 17, 32, 33])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_few_rows_and_many_columns(b200s, m, bias, residual):
    """Generated tokens against a wide layer, with and without bias and residual; 4096 columns of 1024 elements end where
    their allocation does."""
    x, w, b, r, dy = inputs(m, 1024, 4096, torch.bfloat16, bias, residual)
    for act in ("none", "gelu"):
        run_case(b200s, x, w, b, r, act, dy if m == 17 else None)


@pytest.mark.parametrize("m", [1, 9, 40, 257])
def test_strides_and_offsets(b200s, m):
    """x, weight, residual and the gradient as slices of wider tensors, off 16-byte boundaries and transposed."""
    k, n = 264, 200
    x, w, b, r, dy = inputs(m, k, n, torch.bfloat16)

    def inside(t, left, right):
        wide = torch.full((t.shape[0], t.shape[1] + left + right), float("nan"), device="cuda", dtype=t.dtype)
        wide[:, left:left + t.shape[1]] = t
        return wide[:, left:left + t.shape[1]]

    for left, right in ((8, 8), (1, 2)):
        run_case(b200s, inside(x, left, right), inside(w, left, right), b, inside(r, left, right), "silu", inside(dy, left, right))
    tr = lambda t: t.t().contiguous().t()  # noqa: E731
    run_case(b200s, tr(x), tr(w), b, tr(r), "silu", tr(dy))
    run_case(b200s, x, w, b, r[:1].expand(m, n), "silu", dy[:, :1].expand(m, n))
    y = b200s.linear_act(x.view(1, m, k), w, b, "silu", r.view(1, m, n))
    assert y.shape == (1, m, n) and torch.equal(y[0], b200s.linear_act(x, w, b, "silu", r))


@pytest.mark.parametrize("algo,depth", [("classic", 1), ("classic", 2), ("winograd", 1), ("classic", 3), ("auto", -1)])
def test_other_algorithms(b200s, algo, depth):
    """The epilogue behind a Strassen product: the same call with the product's own error, which is compared
    with that of the plain product (operand sums are rounded, so the bound above does not apply)."""
    x, w, b, r, dy = inputs(512, 512, 256, torch.bfloat16)
    plain = b200s.matmul(x, w.t(), algo=algo, depth=depth, out_dtype=torch.float32)
    z = plain.double() + b.double()
    y = act64(z, "gelu") + r.double()
    # one-pass and pipelined recombinations of the same products differ by fp32 roundings only (below 2^-18 here)
    check("y", b200s.linear_act(x, w, b, "gelu", r, algo=algo, depth=depth), y, 2.0 ** -17 * (1 + z.abs() + y.abs()), torch.bfloat16)
    xg = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(b200s.linear_act(xg, w, b, "gelu", r, algo=algo, depth=depth), xg, dy)
    ref = (dy.double() * dact64(z, "gelu")) @ w.double()
    assert ((dx.double() - ref).norm() / ref.norm()).item() < 2.5e-2     # the two-level error of the parity tests


def test_masked_infinite_and_nan_values(b200s):
    """Infinities and NaN stay in their rows; relu and relu2 of NaN are NaN; -inf through gelu's tail is not a number
    as in the formula z * Phi(z), and large negative values give zero."""
    x, w, b, _, _ = inputs(20, 64, 48, torch.float32, residual=False)
    clean = b200s.linear_act(x, w, b, "gelu", precision="tf32")
    x2 = x.clone()
    x2[3, 5] = float("nan")
    x2[19, 0] = float("inf")
    for act in ACTS:
        y = b200s.linear_act(x2, w, b, act, precision="tf32")
        keep = [i for i in range(20) if i not in (3, 19)]
        assert torch.isfinite(y[keep]).all() and torch.isnan(y[3]).all()
    assert torch.equal(b200s.linear_act(x2, w, b, "gelu", precision="tf32")[keep], clean[keep])
    big = torch.full((1, 8), -1e4, device="cuda", dtype=torch.bfloat16)
    for act in ("relu", "relu2", "silu", "gelu", "gelu_tanh"):
        assert not b200s.linear_act(big, torch.ones(8, 8, device="cuda", dtype=torch.bfloat16), None, act).any()


def test_gradient_against_differences(b200s):
    """Central differences of the 64-bit formula; the fp32 gradient is good to 2^-14 of its terms here (three TF32
    passes: 1e-5 of a product, twice)."""
    x, w, b, r, dy = inputs(5, 12, 8, torch.float32)
    for act in ("gelu", "silu", "relu2", "gelu_tanh"):
        v = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        grads = torch.autograd.grad(b200s.linear_act(*v[:3], act, v[3]), v, dy)
        f = lambda x, w, b, r: ((act64(x @ w.t() + b, act) + r) * dy.double()).sum()  # noqa: E731
        args, h = [t.double() for t in (x, w, b, r)], 1e-6
        for k, grad in enumerate(grads):
            for at in (0, grad.numel() // 2, grad.numel() - 1):
                lo, hi = [a.clone() for a in args], [a.clone() for a in args]
                lo[k].view(-1)[at] -= h
                hi[k].view(-1)[at] += h
                diff = ((f(*hi) - f(*lo)) / (2 * h)).item()
                assert abs(grad.reshape(-1)[at].item() - diff) < 2.0 ** -14 * (10 + abs(diff))


def test_empty_batch(b200s):
    x, w, b, r, dy = inputs(4, 64, 48, torch.bfloat16)
    v = [x[:0].clone().requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y = b200s.linear_act(*v, "gelu", r[:0])
    dx, dw, db = torch.autograd.grad(y, v, dy[:0])
    assert y.shape == (0, 48) and dx.shape == (0, 64) and not dw.any() and not db.any()


@pytest.mark.parametrize("m", [2, 300])
def test_graphs_streams_and_repeats(b200s, m):
    """Two captured graphs with their own workspaces replayed one after the other and on two streams at once give what
    eager calls give, bit for bit."""
    x, w, b, r, dy = inputs(m, 768, 640, torch.bfloat16)
    xs = [x.clone().requires_grad_(True), x.flip(0).contiguous().requires_grad_(True)]
    wg, bg = w.requires_grad_(True), b.requires_grad_(True)

    def step(xi):
        y = b200s.linear_act(xi, wg, bg, "gelu", r)
        return (y.detach(),) + torch.autograd.grad(y, (xi, wg, bg), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(xi) for xi in xs]
        again = [step(xi) for xi in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for a, c in zip(want, again) for p, q in zip(a, c))
    graphs, outs = [], []
    for xi in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(xi))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    for a, c in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_two_threads_on_one_stream(b200s):
    """Calls from two host threads share the stream and the allocator: each keeps its own scratch and results."""
    import threading

    cases = [inputs(300, 515, 770, torch.bfloat16, seed=s) for s in (1, 2)]

    def step(c):
        x, w, b, r, dy = c
        v = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = b200s.linear_act(*v, "gelu", r)
        return [y.detach()] + list(torch.autograd.grad(y, v, dy))

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        for _ in range(40):
            got = step(cases[k])
            if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_offsets_past_32_bits(b200s):
    """A result of more than 2^31 elements (4.3 GB), stored by TMA and, with rows of odd length, element by element."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for m, n in ((66000, 32768), (70001, 31003)):
        x = torch.zeros(m, 16, device="cuda", dtype=torch.bfloat16)
        x[-3:] = torch.randn(3, 16, generator=g, device="cuda").bfloat16()
        w = torch.randn(n, 16, generator=g, device="cuda").bfloat16()
        y = b200s.linear_act(x, w, None, "silu")
        want = act64(x[-3:].double() @ w.double().t(), "silu")
        check("last rows", y[-3:], want, 2.0 ** -15 * (1 + want.abs()), torch.bfloat16)
        assert not y[-200:-3].any()
        del y


def test_the_table_decides_between_dense_and_strassen(b200s, tmp_path):
    """algo "auto" follows the tuner table at every call: dense entries give the dense layer bit for bit, a Strassen
    entry the Strassen product."""
    from strassen_triton_b200 import _lib

    lib = _lib.load()
    keep = str(tmp_path / "table.txt").encode()
    assert lib.b200s_tuner_save(keep) == 0
    x, w, b, r, _ = inputs(512, 512, 512, torch.bfloat16)
    dense = b200s.linear_act(x, w, b, "gelu", r)
    strassen = b200s.linear_act(x, w, b, "gelu", r, algo="classic", depth=1)
    try:
        for algo, depth, want in ((_lib.ALGO_DENSE, 0, dense), (_lib.ALGO_CLASSIC, 1, strassen), (_lib.ALGO_DENSE, 0, dense)):
            lib.b200s_tuner_clear()
            assert lib.b200s_tuner_record(512, 512, 512, _lib.BF16, algo, depth) == 0
            assert torch.equal(b200s.linear_act(x, w, b, "gelu", r, algo="auto", depth=-1), want)
    finally:
        lib.b200s_tuner_clear()
        assert lib.b200s_tuner_load(keep) == 0
    assert not torch.equal(dense, strassen)


def test_linear_strassen_module(b200s):
    """LinearStrassen's activation and residual, and the plain layer left as it was."""
    from model.layers import LinearStrassen

    torch.manual_seed(3)
    layer = LinearStrassen(256, 384, bias=True, dtype=torch.bfloat16, depth=0, device="cuda", activation="relu2")
    x = torch.randn(2, 50, 256, device="cuda", dtype=torch.bfloat16)
    res = torch.randn(2, 50, 384, device="cuda", dtype=torch.bfloat16)
    y = layer(x, residual=res)
    assert y.shape == (2, 50, 384)
    assert torch.equal(y, b200s.linear_act(x, layer.weight, layer.bias, "relu2", res))
    plain = LinearStrassen(256, 384, bias=True, dtype=torch.bfloat16, depth=0, device="cuda")
    plain.load_state_dict(layer.state_dict())
    from strassen_triton_b200 import ops
    assert torch.equal(plain(x).view(100, 384), ops.matmul(x.view(100, 256), plain.weight.t(), algo="dense", bias=plain.bias))
    with pytest.raises(ValueError):
        LinearStrassen(8, 8, activation="tanh")


def test_unknown_precision_is_refused_on_every_path(b200s):
    for dtype in (torch.bfloat16, torch.float32):
        x, w = torch.ones(4, 16, device="cuda", dtype=dtype), torch.ones(8, 16, device="cuda", dtype=dtype)
        with pytest.raises(ValueError, match="precision"):
            b200s.linear_act(x, w, precision="fp8")
        assert torch.equal(b200s.linear_act(x, w, precision="tf32"), torch.full((4, 8), 16.0, device="cuda", dtype=dtype))
