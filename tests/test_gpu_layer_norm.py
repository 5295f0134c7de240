"""Layer norm forward and backward against its formula in 64 bits.

Tolerances, elementwise. Results are rounded once: half a step, eps(T)/2 of the value (and half the smallest
subnormal). Before that everything is fp32 with sums whose longest chain of additions is
c = d / 32 + 40 (a thread's share of the row, the warp's and the block's trees), each addition within
2^-24 of the running value, so a mean carries c * 2^-24 of the mean absolute value.
"""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def b200s(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    import strassen_triton_b200

    return strassen_triton_b200


def half_step(ref, dtype):
    return ref.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def reference(x, w, b, eps, dy=None):
    """All results and their tolerances before rounding, in 64 bits."""
    x, w, b = x.double(), w.double(), b.double()
    d, rows = x.shape[1], x.shape[0]
    mu = x.mean(1, keepdim=True)
    var = (x - mu).square().mean(1, keepdim=True)
    rs = (var + eps).rsqrt()
    xh = (x - mu) * rs
    c = d / 32 + 40
    e_mu = c * U * x.abs().mean(1, keepdim=True) + U * mu.abs()
    # rstd: c roundings of the mean square, and the mean's error (second order in it), plus the operations themselves
    e_rs = rs * ((c / 2 + 4) * U + (e_mu * rs) ** 2)
    e_xh = rs * e_mu + xh.abs() * e_rs / rs + 3 * U * (xh.abs() + (x.abs() + mu.abs()) * rs)
    out = {"y": (xh * w + b, e_xh * w.abs() + 2 * U * ((xh * w).abs() + b.abs()))}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    a1, a2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    e_m2 = (c + 4) * U * a2 + (g.abs() * e_xh).mean(1, keepdim=True)
    dx = rs * (g - m1 - xh * m2)
    e_dx = rs * (2 * U * g.abs() + (c + 2) * U * a1 + xh.abs() * e_m2 + e_xh * m2.abs() + 4 * U * (g.abs() + a1 + (xh * m2).abs()))
    e_dx = e_dx + dx.abs() * (e_rs / rs)
    out["dx"] = (dx, e_dx)
    chain = rows / 32 + 200          # a thread's share of the rows, its block's tree, the partial sums
    out["dw"] = ((dy * xh).sum(0), (dy.abs() * e_xh).sum(0) + chain * U * (dy * xh).abs().sum(0))
    out["db"] = (dy.sum(0), chain * U * dy.abs().sum(0))
    return out


def check(name, got, want, dtype):
    ref, tol = want
    tol = tol * 1.01 + half_step(ref.abs() + tol, dtype)
    err = (got.double() - ref).abs()
    assert got.dtype == dtype
    worst = (err / tol.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: error is {worst:.2f} of the tolerance"


def inputs(rows, d, dtype, wdtype, seed=0, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 131 + d)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (r(rows, d) * (1 + 7 * (torch.rand(d, generator=g, device="cuda") < 0.02)) + shift * r(rows, 1)).to(dtype)
    return x, (1 + 0.1 * r(d)).to(wdtype), (0.1 * r(d)).to(wdtype), r(rows, d).to(dtype)


SHAPES = [(700, 2048), (500, 5000), (310, 16384), (460, 4096), (20, 20000), (900, 1030), (1, 1), (1, 768), (3, 7), (5, 33), (2, 255), (64, 256), (37, 768), (300, 1024), (9, 1601), (33, 4096), (8, 4104),
          (5, 8192), (3, 12289), (2, 40000), (1000, 64), (2049, 48), (1, 2), (17, 96), (130, 2304)]


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                          (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_forward_and_backward(b200s, rows, d, dtype, wdtype):
    x, w, b, dy = inputs(rows, d, dtype, wdtype)
    want = reference(x, w, b, 1e-5, dy)
    check("y without gradients", b200s.layer_norm(x, w, b), want["y"], dtype)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = b200s.layer_norm(x, w, b)
    check("y", y.detach(), want["y"], dtype)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    check("dx", dx, want["dx"], dtype)
    check("dw", dw, want["dw"], wdtype)
    check("db", db, want["db"], wdtype)
    assert torch.equal(dx, torch.autograd.grad(b200s.layer_norm(x, w, b), x, dy)[0])     # same call, same bits


@pytest.mark.parametrize("d", [5, 64, 768, 1601])
def test_strides_offsets_and_missing_parameters(b200s, d):
    """Rows of a wider matrix, rows off every alignment, repeated rows, 3-D views, a transposed gradient."""
    x, w, b, dy = inputs(24, d, torch.bfloat16, torch.bfloat16)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    wide = torch.zeros(24, d + 3, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:1 + d] = x
    before = wide.clone()
    view = wide[:, 1:1 + d]
    check("offset rows", b200s.layer_norm(view, w, b), reference(x, w, b, 1e-5)["y"], torch.bfloat16)
    assert torch.equal(wide, before)
    check("3-D", b200s.layer_norm(view.view(4, 6, d) if d + 3 == d else view.reshape(4, 6, d), w, b).reshape(24, d),
          reference(x, w, b, 1e-5)["y"], torch.bfloat16)
    same = x[:1].expand(24, d)
    check("repeated rows", b200s.layer_norm(same, w, b), reference(same, w, b, 1e-5)["y"], torch.bfloat16)
    check("no weight", b200s.layer_norm(x, None, b), reference(x, one, b, 1e-5)["y"], torch.bfloat16)
    check("no bias", b200s.layer_norm(x, w), reference(x, w, zero, 1e-5)["y"], torch.bfloat16)
    xg = x.clone().requires_grad_(True)
    dyt = dy.t().contiguous().t()                 # columns contiguous
    dx, = torch.autograd.grad(b200s.layer_norm(xg), xg, dyt)
    check("dx without parameters", dx, reference(x, one, zero, 1e-5, dy)["dx"], torch.bfloat16)
    wg = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(b200s.layer_norm(view, wg, b), wg, dy[:1].expand(24, d))
    check("dw only", dw, reference(x, w, b, 1e-5, dy[:1].expand(24, d))["dw"], torch.bfloat16)
    bg = b.clone().requires_grad_(True)
    db, = torch.autograd.grad(b200s.layer_norm(view, None, bg), bg, dy)
    check("db only", db, reference(x, one, b, 1e-5, dy)["db"], torch.bfloat16)


def test_constant_rows_far_from_zero_and_nan(b200s):
    """Variance is taken around the mean: a row of equal values gives zeros, not noise; a NaN stays in its row."""
    x = torch.full((4, 1024), 1000.0, device="cuda")
    x[1] += torch.arange(1024, device="cuda") % 2       # 1000, 1001, ...: variance 1/4
    y = b200s.layer_norm(x, None, None)
    assert y[0].abs().max() < 1e-1 and torch.allclose(y[1].abs(), torch.full_like(y[1], 0.25 / (0.25 + 1e-5)).sqrt(), atol=1e-3)
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    y = b200s.layer_norm(x, None, None)
    assert torch.isfinite(y[:2]).all() and torch.isnan(y[2]).all() and torch.isnan(y[3]).any()


def test_empty_batches(b200s):
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = b200s.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and not dw.any() and not db.any()


def test_gradient_against_differences(b200s):
    x, w, b, dy = inputs(3, 40, torch.float32, torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    dx, dw, db = torch.autograd.grad(b200s.layer_norm(x, w, b), (x, w, b), dy)
    f = lambda x, w, b: (torch.nn.functional.layer_norm(x, (40,), w, b) * dy.double()).sum()  # noqa: E731
    args = [t.detach().double() for t in (x, w, b)]
    h = 1e-6
    for k, grad in ((0, dx), (1, dw), (2, db)):
        for at in (0, 17, grad.numel() - 1):
            lo, hi = [a.clone() for a in args], [a.clone() for a in args]
            lo[k].view(-1)[at] -= h
            hi[k].view(-1)[at] += h
            diff = (f(*hi) - f(*lo)) / (2 * h)
            # central differences in 64 bits are good to about h^2 + 1e-16/h; the kernel to 2^-18 of the terms' size (< 20)
            assert abs(grad.reshape(-1)[at].item() - diff.item()) < 20 * 2.0 ** -18


def test_module_graph_and_side_stream(b200s):
    """The module keeps nn.LayerNorm's state; a captured forward and backward replays on new values; a call on
    another stream than the default uses that stream."""
    m = b200s.LayerNorm(768, dtype=torch.bfloat16)
    m.load_state_dict(torch.nn.LayerNorm(768, dtype=torch.bfloat16).state_dict())
    x, w, b, dy = inputs(50, 768, torch.bfloat16, torch.bfloat16)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    check("module", m(x).detach(), reference(x, w, b, 1e-5)["y"], torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    xs = x.clone().requires_grad_(True)
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(m(xs), (xs, m.weight, m.bias), dy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(xs)
        grads = torch.autograd.grad(y, (xs, m.weight, m.bias), dy)
    x2, _, _, dy2 = inputs(50, 768, torch.bfloat16, torch.bfloat16, seed=9)
    with torch.no_grad():
        xs.copy_(x2)
        dy.copy_(dy2)
    g.replay()
    want = reference(x2, w, b, 1e-5, dy2)
    check("replayed y", y.detach(), want["y"], torch.bfloat16)
    for name, got in zip(("dx", "dw", "db"), grads):
        check("replayed " + name, got, want[name], torch.bfloat16)


def test_long_batch_offsets_past_32_bits(b200s):
    """More than 2^31 elements: the last rows are right too (a 16-bit matrix of 4.3 GB, forward and dx)."""
    rows, d = (1 << 31) // 4096 + 5, 4096
    x = torch.empty(rows, d, device="cuda", dtype=torch.bfloat16)
    tail, w, b, dy = inputs(6, d, torch.bfloat16, torch.bfloat16)
    x.zero_()
    x[-6:] = tail
    x.requires_grad_(True)
    y = b200s.layer_norm(x, w, b)
    want = reference(tail, w, b, 1e-5, dy)
    check("last rows", y[-6:].detach(), want["y"], torch.bfloat16)
    g = torch.zeros_like(y)
    g[-6:] = dy
    dx, = torch.autograd.grad(y, x, g)
    check("last rows' dx", dx[-6:], want["dx"], torch.bfloat16)
    assert not dx[:-6].any()


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHILD = r"""
import sys, torch
sys.path.insert(0, %r)
import strassen_triton_b200 as b200s
from tests.test_gpu_layer_norm import check, inputs, reference
for rows, d, dtype in ((500, 3056, torch.bfloat16), (500, 3064, torch.float16), (700, 1528, torch.bfloat16),
                       (700, 1744, torch.float16), (700, 1224, torch.float32)):
    x, w, b, dy = inputs(rows, d, dtype, dtype)
    want = reference(x, w, b, 1e-5, dy)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = b200s.layer_norm(x, w, b)
    check("y", y.detach(), want["y"], dtype)
    for name, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)):
        check(name, got, want[name], dtype)
print("rows ok")
""" % ROOT


def test_row_lengths_whose_ring_just_fits_without_opting_in(built_library):
    """Rings of 48 KB less a little: with the kernels' own shared memory they are above what a launch gets unasked. In a
    process of its own, because a longer row before them raises the limit of the kernel they share."""
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    out = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and "rows ok" in out.stdout, out.stdout[-2000:] + out.stderr[-4000:]
