"""The training-step operators in a run: the GPT-2 model with its norms, epilogues and loss on the library, its
gradients and their clipping, and all of them inside a traced graph."""
import math
import os
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def gpt(built_library):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    from strassen_triton_b200 import fsdp_gpt2

    return fsdp_gpt2


def loss_of(model, idx, targets, vocab):
    """The unfused model's loss over the real columns, in the model's own precision up to the logits."""
    x = model.wte(idx) + model.wpe(torch.arange(idx.shape[1], device=idx.device))
    for blk in model.blocks:
        x = blk(x)
    logits = model.lm_head(model.ln_f(x))[..., :vocab]
    logits = logits if logits.dtype == torch.float64 else logits.float()
    return F.cross_entropy(logits.reshape(-1, vocab), targets.reshape(-1))


def grads_of(model):
    return {n: p.grad.detach().double() for n, p in model.named_parameters()}


def test_fused_model_gradients(gpt):
    """Same bf16 weights in three models: fused, plain torch layers, and plain in 64 bits as the truth. The fused step
    rounds less often than the plain one (residual sums, activations and the loss stay fp32 until stored), so its
    error may exceed the plain one's by the luck of roundings only: 1.5 times, and 2e-3 for parameters whose
    plain error happens to be small."""
    torch.manual_seed(11)
    cfg = dict(layers=2, d=256, heads=4, seq=128)
    base = gpt.GPT(**cfg, device="cuda", plain=True).to(torch.bfloat16)
    state = {k: v.clone() for k, v in base.state_dict().items()}
    fused = gpt.GPT(**cfg, device="cuda", fused=True).to(torch.bfloat16)
    fused.load_state_dict(state)
    exact = gpt.GPT(**cfg, device="cuda", plain=True).double()
    exact.load_state_dict({k: v.double() for k, v in state.items()})
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(0, gpt.VOCAB, (3, 129), generator=g, device="cuda")
    idx, targets = ids[:, :-1], ids[:, 1:].clone()
    targets[0, :20] = -100
    losses = {}
    for name, model in (("plain", base), ("exact", exact)):
        loss = loss_of(model, idx, targets, gpt.VOCAB)
        loss.backward()
        losses[name] = loss.item()
    loss = fused(idx, targets)
    loss.backward()
    losses["fused"] = loss.item()
    assert abs(losses["fused"] - losses["exact"]) < 1e-2       # bf16 logits of size ~1, averaged over 364 tokens
    ref, ours, plain = grads_of(exact), grads_of(fused), grads_of(base)
    for n in ref:
        e = lambda t: ((t - ref[n]).norm() / ref[n].norm().clamp_min(1e-30)).item()  # noqa: E731
        assert e(ours[n]) <= 1.5 * e(plain[n]) + 2e-3, (n, e(ours[n]), e(plain[n]))


def test_train_steps_with_clipping(gpt):
    """The command's loop with every operator: steps run, gradients are finite, and the clipped norm is the bound."""
    torch.manual_seed(1)
    model = gpt.build(layers=1, seq=64, depth=None, device="cuda", world=0, fused=True)
    losses = gpt.train_steps(model, 2, batch=2, seq=64, rank=0, clip=0.05)
    assert all(math.isfinite(x) for x in losses)
    ids = torch.randint(0, gpt.VOCAB, (2, 65), device="cuda")
    model(ids[:, :-1], ids[:, 1:]).backward()
    from strassen_triton_b200 import clip_grad_norm_, grad_norm

    grads = [p.grad for p in model.parameters()]
    before = [t.clone() for t in grads]
    norm = clip_grad_norm_(model.parameters(), 0.05)
    want = math.sqrt(sum(t.double().square().sum().item() for t in before))
    assert abs(norm.item() / want - 1) < 2.0 ** -22 and want > 0.05
    # bf16 roundings of the scaled values average out over 10^7 of them: far inside half a step
    assert abs(grad_norm(grads).item() / 0.05 - 1) < 2.0 ** -9
    plain = gpt.build(layers=1, seq=64, depth=None, device="cuda", world=0)
    assert all(math.isfinite(x) for x in gpt.train_steps(plain, 1, batch=2, seq=64, rank=0))


CHILD = r"""
import sys, torch
sys.path.insert(0, %r)
import strassen_triton_b200 as b200s
torch.manual_seed(0)
w = (0.05 * torch.randn(512, 256, device="cuda")).bfloat16().requires_grad_(True)
head = (0.05 * torch.randn(1000, 512, device="cuda")).bfloat16().requires_grad_(True)
b = torch.randn(512, device="cuda").bfloat16().requires_grad_(True)
n1 = b200s.LayerNorm(256, dtype=torch.bfloat16)
x0 = torch.randn(96, 256, device="cuda").bfloat16()
t = torch.randint(0, 1000, (96,), device="cuda")
def step(x):
    h = b200s.linear_act(n1(x), w, b, "gelu")
    h = b200s.linear_act(h, head, None, "none", None)
    r = b200s.token_logprobs(h, t, entropy=True, top_k=3)
    return -r.logprob.mean() + 0.01 * r.entropy.mean() + b200s.cross_entropy(h, t), r.top_ids
def run(f):
    x = x0.clone().requires_grad_(True)
    loss, ids = f(x)
    return (loss.detach(), ids) + torch.autograd.grad(loss, (x, w, b, head, n1.weight, n1.bias))
eager = run(step)
compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
for got in (run(compiled), run(compiled)):
    for a, c in zip(eager, got):
        assert torch.equal(a, c), (a - c).abs().max()
for name, args in (("layer_norm", (x0, n1.weight.detach(), n1.bias.detach(), 1e-5)),
                   ("linear_act", (x0, w.detach(), b.detach(), None, 4, "dense", 0, "")),
                   ("token_logprobs", (x0, t %% 256, 256, -100, True, 3))):
    torch.library.opcheck(getattr(torch.ops.b200s, name).default, args)
print("compiled ok")
""" % ROOT


def test_operators_in_a_traced_graph(built_library):
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    env = {k: v for k, v in os.environ.items() if k != "TORCHDYNAMO_DISABLE"}
    out = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-4000:]
    assert "compiled ok" in out.stdout


def test_another_device_than_the_current_one(built_library):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    import strassen_triton_b200 as b200s

    x = torch.randn(20, 64, device="cuda:1", dtype=torch.bfloat16)
    w = torch.randn(48, 64, device="cuda:1", dtype=torch.bfloat16)
    assert b200s.layer_norm(x).device.index == 1 and b200s.linear_act(x, w).device.index == 1
    assert b200s.grad_norm([x, w]).device.index == 1 and torch.cuda.current_device() == 0
    with pytest.raises(ValueError):
        b200s.linear_act(x, w.to("cuda:0"))
