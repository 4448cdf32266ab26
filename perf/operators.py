"""The head over many positions, as cases to be timed and compared: the cross entropy of hidden rows
against a head's rows without keeping the logits, its gradients, and the product in 8-bit integers
with a scale for each token and channel, with the rounding to 8 bits that goes before it.

Sizes are those of the repository's own workloads (the head of 151936 rows of 1024, prompts of 16,
128, 1000 and 1920 ids, a user's turn of 61, the layers' products) and generic ones between them.
Where ``own`` is false everything is computed in elementary torch operations in 32 bits; where it
is true by the ops of qwen_megakernel_C and lm_head_loss, as a program calls them.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "qwen0.6b_amd")

H, V = 1024, 151936
IGNORE = -100
DTYPES = dict(f16=torch.float16, bf16=torch.bfloat16)


def _engine():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import Qwen06B_architecture as qa

    return qa


def listed():
    return [
        # the log-probability of one next token, from the hidden state a decode step leaves
        dict(name="score_1", kind="score", dtype="f16", t=1, v=V, h=H, ignored=0.0),
        # scoring a user's turn
        dict(name="score_61", kind="score", dtype="f16", t=61, v=V, h=H, ignored=0.0),
        # perplexity of a page, and of the longest prompt
        dict(name="score_999", kind="score", dtype="f16", t=999, v=V, h=H, ignored=0.0),
        dict(name="score_1919", kind="score", dtype="f16", t=1919, v=V, h=H, ignored=0.0),
        # a small model's step: odd vocabulary, rows that are no whole number of tiles, padding
        dict(name="train_77_odd", kind="train", dtype="bf16", t=77, v=30011, h=584, ignored=0.3, grads="both"),
        # something trained in front of a frozen head (an adapter, a prompt's vectors): prompt masked out
        dict(name="train_999_frozen", kind="train", dtype="f16", t=999, v=V, h=H, ignored=0.25, grads="hidden"),
        # the head trained on hidden rows of four contexts of 1024
        dict(name="train_4096", kind="train", dtype="bf16", t=4096, v=V, h=H, ignored=0.0, grads="both"),
        # the head's rows to 8 bits, once per model
        dict(name="quantize_head", kind="quantize", dtype="f16", t=V, h=H),
        # a paragraph's attention outputs to 8 bits
        dict(name="quantize_127", kind="quantize", dtype="bf16", t=127, h=2 * H),
        # one token's logits from the 8-bit head
        dict(name="linear8_1", kind="linear8", dtype="f16", t=1, v=V, h=H),
        # the q, k and v products of a paragraph
        dict(name="linear8_127", kind="linear8", dtype="bf16", t=127, v=4096, h=H),
        # logits of every position of the longest prompt
        dict(name="linear8_1919", kind="linear8", dtype="f16", t=1919, v=V, h=H),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "score", "train", "train", "linear8", "linear8", "quantize"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "quantize":
        return dict(kind=kind, dtype=dtype, t=_log_int(rng, 1, V), h=rng.choice([H, 16 * _log_int(rng, 4, 128)]))
    t = _log_int(rng, 1, 4096 if kind == "train" else 2048)
    v = rng.choice([V, _log_int(rng, 1000, V)])
    if kind == "linear8":
        return dict(kind=kind, dtype=dtype, t=t, v=v, h=rng.choice([H, 16 * _log_int(rng, 4, 64)]))
    c = dict(kind=kind, dtype=dtype, t=t, v=v, h=rng.choice([H, 8 * _log_int(rng, 8, 128)]),
             ignored=rng.choice([0.0, 0.0, 0.3]))
    if kind == "train":
        c["grads"] = rng.choice(["both", "both", "hidden", "weight"])
    return c


# ---- inputs ---------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, t, h = DTYPES[case["dtype"]], case["t"], case["h"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g).mul_(std)

    kind = case["kind"]
    if kind == "quantize":
        # rows of unlike size, a few channels much larger than the others, as activations have them
        x = normal(t, h) * torch.exp(torch.randn(t, 1, device="cuda", generator=g)).to(dtype)
        x[:, torch.randint(0, h, (max(1, h // 200),), device="cuda", generator=g)] *= 8.0
        return dict(case=case, x=x)
    w = normal(case["v"], h, std=1.2 / math.sqrt(h))
    if kind == "linear8":
        x = normal(t, h)
        x[:, torch.randint(0, h, (max(1, h // 200),), device="cuda", generator=g)] *= 8.0
        q, scale = _quantize(w)
        return dict(case=case, x=x, w=q.to(torch.int8), w_scale=scale)
    # Hidden rows lean towards their target's row, by amounts from nothing to a great deal: the model
    # is sure of some targets, surprised by others.
    targets = torch.randint(0, case["v"], (t,), device="cuda", generator=g)
    lean = 12.0 * torch.rand(t, 1, device="cuda", generator=g)
    hidden = (normal(t, h).float() + lean * w[targets].float()).to(dtype)
    # positions that do not count; the first always does, so that the mean has a denominator
    drop = torch.rand(t, device="cuda", generator=g) < case["ignored"]
    drop[0] = False
    targets = torch.where(drop, torch.full_like(targets, IGNORE), targets)
    s = dict(case=case, hidden=hidden, w=w, targets=targets)
    if kind == "train":
        # fp16 gradients of a mean over thousands of tokens and a large vocabulary need the loss
        # scaled, as a program that trains in fp16 does
        s["loss_scale"] = 65536.0 if dtype == torch.float16 else 1.0
        if own:
            s["hidden"] = hidden.requires_grad_(case["grads"] != "weight")
            s["w"] = w.requires_grad_(case["grads"] != "hidden")
    return s


# ---- one pass -------------------------------------------------------------------------------


def _quantize(x):
    """Rows to 8 bits: scale = max |x| / 127, q = x 127 / max |x| to the nearest, ties to even."""
    x = x.float()
    top = x.abs().amax(dim=1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(top > 0, top, torch.ones_like(top)))
    return q, (top / 127.0).squeeze(1)


def _head(hidden, w, targets):
    """Loss and log of the sum of exponentials of every row, with the logits they came from."""
    logits = hidden.float() @ w.float().t()
    top = logits.amax(dim=1, keepdim=True)
    lse = (top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))).squeeze(1)
    counts = targets != IGNORE
    at = torch.where(counts, targets, torch.zeros_like(targets))
    loss = lse - logits.gather(1, at[:, None]).squeeze(1)
    return torch.where(counts, loss, torch.zeros_like(loss)), lse, logits, counts, at


def _train(s):
    hidden, w, grads = s["hidden"], s["w"], s["case"]["grads"]
    loss, lse, logits, counts, at = _head(hidden, w, s["targets"])
    n = counts.sum().float()
    p = torch.exp(logits - lse[:, None])
    p[torch.arange(p.shape[0], device=p.device), at] -= 1.0
    p *= torch.where(counts, s["loss_scale"] / n, torch.zeros_like(n))[:, None]
    out = dict(loss=loss.sum() / n * s["loss_scale"])
    if grads != "weight":
        out["grad_hidden"] = (p @ w.float()).to(hidden.dtype)
    if grads != "hidden":
        out["grad_weight"] = (p.t() @ hidden.float()).to(w.dtype)
    return out


def _linear8(s):
    q, scale = _quantize(s["x"])
    w, k = s["w"], q.shape[1]
    # sums of 1024 products of 8-bit numbers are exact in 32-bit floats
    acc = sum(q[:, i:i + 1024].contiguous() @ w[:, i:i + 1024].float().t() for i in range(0, k, 1024))
    return (acc * scale[:, None] * s["w_scale"][None, :]).to(s["x"].dtype)


def _run_own(s):
    kind, qa = s["case"]["kind"], _engine()
    ops = qa.qwen_megakernel_C
    if kind == "score":
        loss, lse = ops.lm_head_cross_entropy(s["hidden"], s["w"], s["targets"])
        return dict(loss=loss, lse=lse)
    if kind == "train":
        hidden, w, grads = s["hidden"], s["w"], s["case"]["grads"]
        loss = qa.lm_head_loss(hidden, w, s["targets"]) * s["loss_scale"]
        leaves = [x for x in (hidden, w) if x.requires_grad]
        got = torch.autograd.grad(loss, leaves)
        names = dict(both=("grad_hidden", "grad_weight"), hidden=("grad_hidden",), weight=("grad_weight",))[grads]
        return dict(loss=loss.detach(), **dict(zip(names, got)))
    if kind == "quantize":
        q, scale = ops.quantize_rows(s["x"])
        return dict(values=q * scale[:, None], scale=scale)
    q, scale = ops.quantize_rows(s["x"])
    return ops.matmul_i8(q, scale, s["w"], s["w_scale"], s["x"].dtype)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "score":
        loss, lse = _head(state["hidden"], state["w"], state["targets"])[:2]
        return dict(loss=loss, lse=lse)
    if kind == "train":
        return _train(state)
    if kind == "quantize":
        q, scale = _quantize(state["x"])
        return dict(values=q * scale[:, None], scale=scale)
    return _linear8(state)


# ---- what it cannot do without --------------------------------------------------------------


def work(case):
    kind, t, h = case["kind"], case["t"], case["h"]
    if kind == "quantize":
        # a 16-bit entry read and its value written (8 bits and a 32-bit scale a row stand for it)
        return dict(bytes=t * h * 3 + 4 * t, flops=2 * t * h)
    v = case["v"]
    if kind == "linear8":
        return dict(bytes=2 * t * h + v * h + 4 * v + 2 * t * v, flops=2 * t * v * h)
    read = 2 * t * h + 2 * v * h + 8 * t
    if kind == "score":
        return dict(bytes=read + 8 * t, flops=2 * t * v * h)
    n_grads = 2 if case["grads"] == "both" else 1
    written = (2 * t * h if case["grads"] != "weight" else 0) + (2 * v * h if case["grads"] != "hidden" else 0)
    return dict(bytes=read + written, flops=2 * t * v * h * (1 + n_grads))


# ---- the definition, in 64 bits -------------------------------------------------------------


def exact(case, seed):
    """From the definitions: rows are taken some at a time, so that 64-bit logits of a long text fit."""
    s = prepare(case, seed)
    kind = case["kind"]
    d = torch.float64
    if kind in ("quantize", "linear8"):
        x = s["x"].to(d)
        top = x.abs().max(dim=1).values
        unit = top / 127
        steps = torch.round(127 * x / top.clamp_min(torch.finfo(d).tiny)[:, None])
        if kind == "quantize":
            return dict(values=steps * unit[:, None], scale=unit)
        wt = s["w"].to(d).t().contiguous() * s["w_scale"].to(d)
        return torch.cat([unit[i:i + 256, None] * (steps[i:i + 256] @ wt) for i in range(0, case["t"], 256)])
    hidden, w, targets = s["hidden"].detach().to(d), s["w"].detach().to(d), s["targets"]
    keep = targets.ne(IGNORE)
    scale = s.get("loss_scale", 1.0) / int(keep.sum())
    losses, lses, gh = [], [], []
    gw = torch.zeros_like(w) if kind == "train" and case["grads"] != "hidden" else None
    wt = w.t().contiguous()
    for i in range(0, case["t"], 256):
        x, y, k = hidden[i:i + 256], targets[i:i + 256], keep[i:i + 256]
        z = x @ wt
        lse = torch.logsumexp(z, dim=1)
        picked = z[torch.arange(len(y), device=z.device), y.clamp_min(0)]
        losses.append((lse - picked) * k)
        lses.append(lse)
        if kind == "train":
            delta = torch.softmax(z, dim=1)
            delta[torch.arange(len(y), device=z.device), y.clamp_min(0)] -= 1
            delta *= (k * scale)[:, None]
            if case["grads"] != "weight":
                gh.append(delta @ w)
            if gw is not None:
                gw += delta.t().contiguous() @ x
    if kind == "score":
        return dict(loss=torch.cat(losses), lse=torch.cat(lses))
    out = dict(loss=torch.cat(losses).sum() * scale)
    if gh:
        out["grad_hidden"] = torch.cat(gh)
    if gw is not None:
        out["grad_weight"] = gw
    return out
