"""Cases of the training-step operators: layer norm, the linear layer with its epilogue, token log
probabilities and gradient clipping, forwards and backwards, from one token to full training batches.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, 64 where a sum is
long) or, with ``own`` set, through the calls a user makes of this package; ``exact`` computes the
same outputs from the operators' definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ACT = ("none", "relu", "relu2", "silu", "gelu", "gelu_tanh")


def listed():
    return [
        # the norm before a block when one sequence generates one token: pure latency
        dict(name="norm_one_token", op="norm", rows=1, d=768, dtype="bf16", wdtype="bf16", train=False),
        # ln1 / ln2 of the GPT-2-124M step: 8 sequences of 1024 tokens
        dict(name="norm_gpt2_train", op="norm", rows=8192, d=768, dtype="bf16", wdtype="bf16", train=True),
        # a wide model with fp32 norm parameters beside 16-bit activations
        dict(name="norm_wide_train", op="norm", rows=16381, d=4096, dtype="fp16", wdtype="fp32", train=True),
        # the qkv projection for one generated token
        dict(name="linear_one_token", op="linear", m=1, k=768, n=2304, dtype="bf16", bias=True, act="none",
             residual=False, train=False),
        # a feed-forward layer of the GPT-2-124M step with its gradients
        dict(name="linear_gelu_train", op="linear", m=8192, k=768, n=2304, dtype="bf16", bias=True, act="gelu",
             residual=False, train=True),
        # a gated-size layer of an odd model on a ragged batch, with the residual stream added
        dict(name="linear_odd_train", op="linear", m=1021, k=771, n=1283, dtype="fp16", bias=True, act="silu",
             residual=True, train=True),
        # prompt processing of a large model
        dict(name="linear_large_forward", op="linear", m=8192, k=4096, n=8192, dtype="fp16", bias=True,
             act="relu2", residual=True, train=False),
        # scoring one step of a batch of 8 generated sequences, with the alternatives shown to the user
        dict(name="logprobs_decode", op="logprobs", rows=8, width=50304, vocab=50257, dtype="bf16", masked=False,
             ignored=0.0, entropy=True, top_k=8, train=False),
        # the loss of the GPT-2-124M step: vocabulary padded to 50304 columns
        dict(name="logprobs_gpt2_train", op="logprobs", rows=8192, width=50304, vocab=50257, dtype="bf16",
             masked=False, ignored=0.05, entropy=False, top_k=0, train=True),
        # a policy-gradient step with an entropy bonus over a vocabulary of odd length, some tokens forbidden
        dict(name="logprobs_entropy_train", op="logprobs", rows=515, width=32003, vocab=32003, dtype="fp32",
             masked=True, ignored=0.2, entropy=True, top_k=5, train=True),
        # a healthy step of a small fp32 model: many small tensors, the norm below the bound
        dict(name="clip_small_step", op="clip", kind="mixed", tensors=60, largest=200000, shape_seed=1,
             dtype="fp32", packed=True, out="", over=False),
        # a step of GPT-2-124M whose norm is over the bound, 16-bit gradients clipped into fp32 ones
        dict(name="clip_gpt2_to_fp32", op="clip", kind="gpt2", tensors=101, largest=0, shape_seed=0,
             dtype="bf16", packed=False, out="fp32", over=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(("norm", "linear", "logprobs", "clip"))
    if op == "norm":
        d = _log(rng, 1, 12288)
        rows = _log(rng, 1, max(1, min(16384, (1 << 26) // d)))
        dt = rng.choice(("bf16", "fp16", "fp32"))
        return dict(op=op, rows=rows, d=d, dtype=dt, wdtype=rng.choice((dt, "fp32")), train=rng.random() < 0.6)
    if op == "linear":
        k, n, m = _log(rng, 8, 8192), _log(rng, 8, 8192), _log(rng, 1, 8192)
        if rng.random() < 0.6:      # most layers have rows of whole 16-byte vectors
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        train = rng.random() < 0.5
        m = max(1, min(m, ((83 if train else 250) << 30) // (k * n)))      # a step has three products instead of one
        return dict(op=op, m=m, k=k, n=n, dtype=rng.choice(("bf16", "fp16")), bias=rng.random() < 0.7,
                    act=rng.choice(_ACT), residual=rng.random() < 0.5, train=train)
    if op == "logprobs":
        vocab = _log(rng, 2, 131072)
        width = vocab if rng.random() < 0.5 else (vocab + 63) // 64 * 64
        dt = rng.choice(("bf16", "fp16", "fp32"))
        rows = _log(rng, 1, max(1, min(8192, (8192 * 50304 // (2 if dt == "fp32" else 1)) // width)))
        few = rows * width <= 1 << 26
        return dict(op=op, rows=rows, width=width, vocab=vocab, dtype=dt, masked=rng.random() < 0.4,
                    ignored=rng.choice((0.0, 0.3)), entropy=rng.random() < 0.5,
                    top_k=min(vocab, rng.choice((0, 1, 5, 20))) if few else 0, train=rng.random() < 0.6)
    out = rng.choice(("", "bf16", "fp32"))
    return dict(op=op, kind="mixed", tensors=_log(rng, 1, 300), largest=_log(rng, 8, 1 << 20),
                shape_seed=rng.randrange(1 << 30), dtype=rng.choice(("bf16", "fp16", "fp32", "any")),
                packed=rng.random() < 0.5, out=out, over=out != "" and rng.random() < 0.7)


def _clip_shapes(case):
    if case["kind"] == "gpt2":
        d, layers, vocab, seq = 768, 12, 50304, 1024
        shapes = [(vocab, d), (seq, d), (d,), (d,), (vocab, d)]
        for _ in range(layers):
            shapes += [(d,), (d,), (d,), (d,), (3 * d, d), (d, d), (4 * d, d), (d, 4 * d)]
        return [(s, case["dtype"]) for s in shapes]
    rng = random.Random(case["shape_seed"])
    out = []
    for _ in range(case["tensors"]):
        n = _log(rng, 1, case["largest"])
        c = _log(rng, 1, n)
        dt = rng.choice(("bf16", "fp16", "fp32")) if case["dtype"] == "any" else case["dtype"]
        out.append(((n // c, c), dt))
    return out


def _clip_layout(case):
    """[(shape, type, first element in the flat buffer of the type)], {type: elements of its buffer}"""
    spans, sizes = [], {}
    for shape, dt in _clip_shapes(case):
        at = sizes.get(dt, 0)
        n = int(np.prod(shape))
        spans.append((shape, dt, at))
        sizes[dt] = at + (n if case["packed"] else (n + 7) // 8 * 8)
    return spans, sizes


def _inputs(case, seed):
    """The tensors of a case, on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "norm":
        dt, wdt, rows, d = _DT[case["dtype"]], _DT[case["wdtype"]], case["rows"], case["d"]
        # a residual stream: a common offset per row and a few columns much larger than the rest
        gain = torch.where(torch.rand(d, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        x = torch.randn((rows, d), generator=g, device="cuda").mul_(gain).add_(randn(rows, 1, scale=0.5)).to(dt)
        s = dict(x=x, w=(1 + randn(d, scale=0.1)).to(wdt), b=randn(d, scale=0.1, dtype=wdt))
        if case["train"]:
            s["dy"] = randn(rows, d, dtype=dt)
        return s
    if case["op"] == "linear":
        dt, m, k, n = _DT[case["dtype"]], case["m"], case["k"], case["n"]
        s = dict(x=randn(m, k, dtype=dt), w=randn(n, k, scale=k ** -0.5, dtype=dt),
                 b=randn(n, scale=0.2, dtype=dt) if case["bias"] else None,
                 r=randn(m, n, dtype=dt) if case["residual"] else None)
        if case["train"]:
            s["dy"] = randn(m, n, dtype=dt)
        return s
    if case["op"] == "logprobs":
        dt, rows, width, vocab = _DT[case["dtype"]], case["rows"], case["width"], case["vocab"]
        logits = torch.randn((rows, width), generator=g, device="cuda").mul_(2.0)
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        # a trained model: the observed token is usually likely
        lift = 6.0 * torch.rand(rows, 1, generator=g, device="cuda")
        logits.scatter_add_(1, targets[:, None], lift)
        logits = logits.to(dt)
        if case["masked"]:
            # forbidden tokens at -inf in one row of two (never the target's); one row keeps the target alone
            forbid = torch.rand((rows, width), generator=g, device="cuda") < 0.3
            forbid[1::2] = False
            forbid[rows // 2] = True
            forbid.scatter_(1, targets[:, None], False)
            logits.masked_fill_(forbid, float("-inf"))
        drop = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        targets = torch.where(drop, torch.full_like(targets, -100), targets)
        s = dict(logits=logits, targets=targets)
        if case["train"]:
            s["dlp"] = randn(rows, scale=1.0 / rows)
            s["dent"] = randn(rows, scale=0.01 / rows) if case["entropy"] else None
        return s
    # gradients as a data-parallel wrapper keeps them: views into one flat buffer per type
    spans, sizes = _clip_layout(case)
    flats = {dt: torch.zeros(n, device="cuda", dtype=_DT[dt]) for dt, n in sizes.items()}
    grads = []
    for i, (shape, dt, at) in enumerate(spans):
        n = int(np.prod(shape))
        view = flats[dt][at:at + n]
        view.copy_(randn(n, scale=1e-3 * (1 + 5 * (i % 7 == 0))))
        grads.append(view.view(shape))
    numel = sum(t.numel() for t in grads)
    # expected norm of the values above is within a few percent of 1e-3 sqrt(numel) .. 6e-3 sqrt(numel)
    return dict(grads=grads, flats=list(flats.values()),
                max_norm=(0.25e-3 if case["over"] else 50e-3) * math.sqrt(numel))


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "clip":
        # gradients below the bound stay where they are; clipped ones go to the optimizer's own flat buffers
        if case["out"]:
            src = s["flats"]
            s["flats"] = [torch.zeros_like(f, dtype=_DT[case["out"]]) for f in src]
            base = {f.dtype: (f, o) for f, o in zip(src, s["flats"])}
            s["out"] = []
            for t in s["grads"]:
                f, o = base[t.dtype]
                at = t.storage_offset()
                s["out"].append(o[at:at + t.numel()].view(t.shape))
        else:
            s["out"] = None
        return s
    if case.get("train"):
        for name in ("x", "w", "b", "r", "logits"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ---- plain forms -------------------------------------------------------------------------------

def _plain_norm(s, eps=1e-5):
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    xf = x.float()
    xc = xf - xf.mean(-1, keepdim=True)
    rstd = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = xc * rstd
    y = (xh * w.float() + b.float()).to(x.dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    gw = dy * w.float()
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dw": (dy * xh).sum(0).to(w.dtype), "db": dy.sum(0).to(b.dtype)}


def _plain_act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "relu2":
        p = z.clamp_min(0)
        return p * p, 2 * p
    if act == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg * (1 + z * (1 - sg))
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(z * -math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    sg = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))       # (1 + tanh u) / 2
    return z * sg, sg + z * sg * (1 - sg) * 2 * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].detach(), s["w"].detach()
    xf, wf = x.float(), w.float()
    z = xf @ wf.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y, da = _plain_act(z, case["act"])
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    y = y.to(x.dtype)
    if not case["train"]:
        return {"y": y}
    dz = s["dy"].float() * da
    out = {"y": y, "dx": (dz @ wf).to(x.dtype), "dw": (dz.t() @ xf).to(w.dtype)}
    if s["b"] is not None:
        out["db"] = dz.sum(0).to(s["b"].dtype)
    if s["r"] is not None:
        out["dr"] = s["dy"].to(s["r"].dtype)
    return out


def _plain_logprobs(s):
    case = s["case"]
    logits, targets, vocab = s["logits"].detach(), s["targets"], case["vocab"]
    x = logits[:, :vocab].float()
    m = x.amax(1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    lp = x - lse
    p = lp.exp()
    ignored = targets == -100
    t = torch.where(ignored, 0, targets)[:, None]
    out = {"logprob": torch.where(ignored, 0.0, lp.gather(1, t)[:, 0])}
    ent = None
    if case["entropy"] or (case["train"] and s["dent"] is not None):
        plp = torch.where(p > 0, p * lp, 0.0)
        ent = -plp.sum(1)
        out["entropy"] = ent
    if case["top_k"]:
        val, idx = torch.sort(x, dim=1, descending=True, stable=True)
        out["top_ids"] = idx[:, :case["top_k"]]
        out["top_logprobs"] = val[:, :case["top_k"]] - lse
    if case["train"]:
        gl = torch.where(ignored, 0.0, s["dlp"])[:, None]
        d = -gl * p
        d.scatter_add_(1, t, gl)
        if s["dent"] is not None:
            d = d - s["dent"][:, None] * (plp + p * ent[:, None])
        full = torch.zeros(logits.shape, dtype=logits.dtype, device=logits.device)
        full[:, :vocab] = d.to(logits.dtype)
        out["dlogits"] = full
    return out


def _plain_clip(s):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in s["grads"]:
        total = total + t.double().square().sum()
    norm = total.sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    if s["out"] is None:
        for t in s["grads"]:
            t.copy_(t.float() * coef)
    else:
        for o, t in zip(s["out"], s["grads"]):
            o.copy_(t.float() * coef)
    return {"norm": norm.float(), "flats": s["flats"]}


# ---- through the package -----------------------------------------------------------------------

def _own(s):
    import strassen_triton_b200 as b200s

    case = s["case"]
    if case["op"] == "norm":
        y = b200s.layer_norm(s["x"], s["w"], s["b"], eps=1e-5)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if case["op"] == "linear":
        y = b200s.linear_act(s["x"], s["w"], s["b"], activation=case["act"], residual=s["r"])
        if not case["train"]:
            return {"y": y}
        names = [k for k in ("x", "w", "b", "r") if s[k] is not None]
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
    if case["op"] == "logprobs":
        r = b200s.token_logprobs(s["logits"], s["targets"], vocab=case["vocab"], ignore_index=-100,
                                 entropy=case["entropy"], top_k=case["top_k"])
        out = {"logprob": r.logprob.detach()}
        if case["entropy"]:
            out["entropy"] = r.entropy.detach()
        if case["top_k"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        if case["train"]:
            outs, gs = [r.logprob], [s["dlp"]]
            if case["entropy"]:
                outs.append(r.entropy)
                gs.append(s["dent"])
            out["dlogits"], = torch.autograd.grad(outs, s["logits"], gs)
        return out
    norm = b200s.clip_grads_(s["grads"], s["max_norm"], out=s["out"])
    return {"norm": norm, "flats": s["flats"]}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "linear": _plain_linear, "logprobs": _plain_logprobs,
                "clip": _plain_clip}[state["case"]["op"]](state)


def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    if case["op"] == "clip":
        es = {"bf16": 2, "fp16": 2, "fp32": 4}
        rd = wr = n = 0
        for shape, dt in _clip_shapes(case):
            k = int(np.prod(shape))
            n += k
            rd += k * es[dt]
            wr += k * es[case["out"]] if case["out"] else 0
        return {"bytes": rd + wr, "flops": 3 * n}
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        e, ws = case["rows"] * case["d"], case["d"] * (4 if case["wdtype"] == "fp32" else 2)
        if case["train"]:
            return {"bytes": 4 * e * es + 4 * ws, "flops": 20 * e}
        return {"bytes": 2 * e * es + 2 * ws, "flops": 8 * e}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        b, r = n * int(case["bias"]), m * n * int(case["residual"])
        nbytes = m * k + n * k + b + r + m * n
        flops = 2 * m * n * k
        if case["train"]:
            nbytes += m * n + m * k + n * k + b
            flops *= 3
        return {"bytes": nbytes * es, "flops": flops}
    e = case["rows"] * case["width"]
    small = case["rows"] * (8 + 4 + 4 * int(case["entropy"]) + 12 * case["top_k"])
    if case["train"]:
        return {"bytes": 2 * e * es + small + 8 * case["rows"], "flops": 10 * e}
    return {"bytes": case["rows"] * case["vocab"] * es + small, "flops": 5 * e}


# ---- definitions in 64 bits --------------------------------------------------------------------

def _act64(z, act):
    F = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: F.relu(z), "relu2": lambda: F.relu(z) ** 2, "silu": lambda: F.silu(z),
            "gelu": lambda: F.gelu(z), "gelu_tanh": lambda: F.gelu(z, approximate="tanh")}[act]()


def _exact_logprobs(case, s):
    parts = {}
    for lo in range(0, case["rows"], 1024):
        hi = min(case["rows"], lo + 1024)
        x = s["logits"][lo:hi, :case["vocab"]].double()
        x.requires_grad_(case["train"])
        t = s["targets"][lo:hi]
        live = torch.isfinite(x.detach())
        # forbidden tokens leave the sums: -1e4 underflows to probability zero in 64 bits
        safe = torch.where(live, x, torch.full_like(x, -1e4))
        lp = torch.log_softmax(safe, 1)
        used = t != -100
        picked = lp[torch.arange(hi - lo, device=t.device), t.clamp_min(0)] * used
        rec = {"logprob": picked.detach()}
        ent = None
        if case["entropy"]:
            ent = -(lp.exp() * lp).sum(1)
            rec["entropy"] = ent.detach()
        if case["top_k"]:
            ids = torch.argsort(x.detach(), dim=1, descending=True, stable=True)[:, :case["top_k"]]
            rec["top_ids"] = ids
            vals = lp.detach().gather(1, ids)
            rec["top_logprobs"] = torch.where(live.gather(1, ids), vals, torch.full_like(vals, float("-inf")))
        if case["train"]:
            loss = (picked * s["dlp"][lo:hi].double()).sum()
            if ent is not None:
                loss = loss + (ent * s["dent"][lo:hi].double()).sum()
            g, = torch.autograd.grad(loss, x)
            rec["dlogits"] = torch.nn.functional.pad(g, (0, case["width"] - case["vocab"]))
        for k, v in rec.items():
            parts.setdefault(k, []).append(v)
    return {k: torch.cat(v) for k, v in parts.items()}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, s)
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(torch.cat([f.double() for f in s["flats"]]))    # what pads the views is zero
        scale = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        return {"norm": norm, "flats": [f.double() * scale for f in s["flats"]]}
    names = [k for k in ("x", "w", "b", "r") if s.get(k) is not None]
    v = {k: s[k].double().requires_grad_(case["train"]) for k in names}
    if case["op"] == "norm":
        y = torch.nn.functional.layer_norm(v["x"], (case["d"],), v["w"], v["b"], 1e-5)
    else:
        y = _act64(torch.nn.functional.linear(v["x"], v["w"], v.get("b")), case["act"])
        if "r" in v:
            y = y + v["r"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [v[k] for k in names], s["dy"].double())
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out
