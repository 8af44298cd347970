"""Measured cases of the operators at the two ends of a token model and of its 8-bit activation
checkpoint: the embedding lookup and its gradient, the softmax cross entropy over the vocabulary with
its gradient, and GEGLU whose backward reads an 8-bit copy of its input.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a training program
holds before the call, run() makes one pass: with `own` false in elementary torch operations in fp32,
with `own` true through this library's public functions.  exact() gives a pass's values in float64.
"""
import importlib
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LIBRARY = Path(__file__).resolve().parent.parent / "kernel-rsi_b200" / "library"
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715


def library(name):
    """A module of the library (its folder goes on sys.path, as its users put it there)."""
    if str(LIBRARY) not in sys.path:
        sys.path.insert(0, str(LIBRARY))
    return importlib.import_module(name)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the rows of one short prompt's 16 tokens, looked up without a gradient: latency
        {"name": "emb_lookup_16", "op": "embedding", "n": 16, "d": 1152, "vocab": 32768, "dtype": "bf16",
         "scale": 1.0, "padding": -1, "step": False},
        # a small fp32 model's step on a half padded batch: odd row width, padding without gradient,
        # the table scaled by sqrt(d)
        {"name": "emb_step_ragged", "op": "embedding", "n": 5003, "d": 250, "vocab": 10007, "dtype": "f32",
         "scale": 15.8, "padding": 0, "step": True},
        # the block model's batch (32 sequences of 1024, d 1152): lookup and the table's gradient
        {"name": "emb_step_32k", "op": "embedding", "n": 32768, "d": 1152, "vocab": 32768, "dtype": "bf16",
         "scale": 1.0, "padding": -1, "step": True},
        # the losses of 16 rows (scoring a short text): the weight's read is all there is
        {"name": "ce_eval_16", "op": "cross_entropy", "n": 16, "d": 768, "vocab": 32768, "dtype": "bf16",
         "scale": 1.0, "z_loss": 0.0, "reduction": "none", "ignored": 0.0, "step": False},
        # a small f16 model's training step, ragged in rows and vocabulary
        {"name": "ce_step_ragged", "op": "cross_entropy", "n": 257, "d": 512, "vocab": 10007, "dtype": "f16",
         "scale": 1.0, "z_loss": 0.0, "reduction": "mean", "ignored": 0.2, "step": True},
        # per-token losses weighted by the caller (its gradient differs from row to row)
        {"name": "ce_step_tokens", "op": "cross_entropy", "n": 2001, "d": 1152, "vocab": 50021, "dtype": "bf16",
         "scale": 1.0, "z_loss": 0.0, "reduction": "none", "ignored": 0.1, "step": True},
        # evaluation with a large multilingual vocabulary
        {"name": "ce_eval_bigvocab", "op": "cross_entropy", "n": 4096, "d": 1024, "vocab": 131072, "dtype": "bf16",
         "scale": 1.0, "z_loss": 0.0, "reduction": "mean", "ignored": 0.0, "step": False},
        # a base-size model's step: tied table (logits scaled by d^-0.5), z-loss, 15% of the rows masked out
        {"name": "ce_step_8k", "op": "cross_entropy", "n": 8192, "d": 768, "vocab": 32768, "dtype": "bf16",
         "scale": 768 ** -0.5, "z_loss": 1e-4, "reduction": "mean", "ignored": 0.15, "step": True},
        # the block model's batch: every one of 32 x 1024 rows has a target
        {"name": "ce_step_32k", "op": "cross_entropy", "n": 32768, "d": 1152, "vocab": 32768, "dtype": "bf16",
         "scale": 1.0, "z_loss": 0.0, "reduction": "mean", "ignored": 0.0, "step": True},
        # GEGLU of one short sequence with its 8-bit checkpoint: latency
        {"name": "geglu8_step_16", "op": "geglu_q8", "n": 16, "d": 4608, "dtype": "bf16"},
        # odd rows, a width that is no multiple of the checkpoint's group, f16
        {"name": "geglu8_step_ragged", "op": "geglu_q8", "n": 1777, "d": 2740, "dtype": "f16"},
        # the block model's feed-forward (FFN 4608) on its whole batch
        {"name": "geglu8_step_32k", "op": "geglu_q8", "n": 32768, "d": 4608, "dtype": "bf16"},
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "cross_entropy", "geglu_q8"])
    if op == "embedding":
        vocab = log_int(rng, 1000, 50021)
        return {"op": op, "n": log_int(rng, 1, 32768), "d": log_int(rng, 64, 1152), "vocab": vocab,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "scale": rng.choice([1.0, 15.8]),
                "padding": rng.choice([-1, 0]), "step": rng.random() < 0.75}
    if op == "cross_entropy":
        vocab = log_int(rng, 1000, 131072)
        d = 8 * log_int(rng, 8, 144)
        return {"op": op, "n": log_int(rng, 1, min(32768, (1 << 30) // vocab)), "d": d, "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "f16"]), "scale": rng.choice([1.0, d ** -0.5]),
                "z_loss": rng.choice([0.0, 1e-4]), "reduction": rng.choice(["mean", "sum", "none"]),
                "ignored": rng.choice([0.0, 0.15]), "step": rng.random() < 0.7}
    return {"op": op, "n": log_int(rng, 1, 32768), "d": log_int(rng, 64, 4608),
            "dtype": rng.choice(["bf16", "f16", "f32"])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    n, d = case["n"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "geglu_q8":
        # a gate|value projection's output: each row at a scale of its own, a few columns far larger
        u = normal(n, 2 * d) * torch.exp(0.5 * normal(n, 1)) * torch.exp(0.7 * normal(1, 2 * d))
        return {"case": case, "u": u.to(dt).requires_grad_(True), "g": normal(n, d).to(dt)}

    v = case["vocab"]
    # token ids as text has them: the probability of an id falls as one over its rank
    ids = (torch.exp(torch.rand(n, generator=g, device="cuda") * math.log(v)) - 1).long().clamp_(0, v - 1)
    if case["op"] == "embedding":
        if case["padding"] >= 0:
            ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, case["padding"], ids)
        return {"case": case, "tokens": ids, "table": normal(v, d).to(dt).requires_grad_(case["step"]),
                "g": normal(n, d).to(dt)}

    # logits of unit noise in which each row's target stands out by 0 to d^0.5 / 2 units
    std = 1.0 if case["scale"] != 1.0 else d ** -0.5
    w = (normal(v, d) * std).to(dt)
    lift = torch.rand(n, 1, generator=g, device="cuda") * (0.5 / std)
    x = (normal(n, d) + lift * w[ids].float()).to(dt)
    targets = torch.where(torch.rand(n, generator=g, device="cuda") < case["ignored"], -100, ids)
    return {"case": case, "x": x.requires_grad_(case["step"]), "w": w.requires_grad_(case["step"]),
            "targets": targets, "g": torch.rand(n, generator=g, device="cuda")}


# ---------------------------------------------------------------- one pass
def run(state):
    return RUN[state["case"]["op"], bool(own)](state)


def embedding_own(s):
    c = s["case"]
    padding = c["padding"] if c["padding"] >= 0 else None
    out = library("embedding").embedding(s["tokens"], s["table"], scale=c["scale"], padding_idx=padding)
    if not c["step"]:
        return out
    return out.detach(), torch.autograd.grad(out, s["table"], s["g"])[0]


def embedding_plain(s):
    c, tokens, table = s["case"], s["tokens"], s["table"].detach()
    out = (table[tokens].float() * c["scale"]).to(table.dtype)
    if not c["step"]:
        return out
    g = s["g"].float() * c["scale"]
    if c["padding"] >= 0:
        g = g * (tokens != c["padding"])[:, None]
    grad = torch.zeros(table.shape, device=table.device).index_add_(0, tokens, g)
    return out, grad.to(table.dtype)


def cross_entropy_own(s):
    c = s["case"]
    loss = library("linear_cross_entropy").linear_cross_entropy(
        s["x"], s["w"], s["targets"], scale=c["scale"], z_loss=c["z_loss"], reduction=c["reduction"])
    if not c["step"]:
        return loss
    up = s["g"] if c["reduction"] == "none" else None
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), up)
    return loss.detach(), dx, dw


def cross_entropy_plain(s):
    c, x, w, targets = s["case"], s["x"].detach(), s["w"].detach(), s["targets"]
    x32, w32 = x.float(), w.float()
    p = (x32 @ w32.t()).mul_(c["scale"])
    keep = targets != -100
    t = torch.where(keep, targets, 0)
    rows = torch.arange(x.shape[0], device=x.device)
    picked = p[rows, t]
    top = p.amax(1, keepdim=True)
    p.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    loss = torch.where(keep, lse - picked + c["z_loss"] * lse * lse, 0.0)
    count = keep.sum().clamp(min=1).float()
    if c["reduction"] == "mean":
        out, up = loss.sum() / count, keep / count
    elif c["reduction"] == "sum":
        out, up = loss.sum(), keep.float()
    else:
        out, up = loss, keep * s["g"]
    if not c["step"]:
        return out
    p.mul_(((1.0 + 2.0 * c["z_loss"] * lse) * up)[:, None] / total)
    p[rows, t] -= up
    p.mul_(c["scale"])
    return out, (p @ w32).to(x.dtype), (p.t() @ x32).to(w.dtype)


def geglu_q8_own(s):
    out = library("geglu_q8").geglu_q8(s["u"])
    return out.detach(), torch.autograd.grad(out, s["u"], s["g"])[0]


def quantised(h):
    """The 8-bit values of one half of the rows and the steps they stand for: groups of 32 columns, the step a
    power of two, 2^-6 of the largest magnitude's leading power (2^-126 at least)."""
    n, d = h.shape
    pad = torch.nn.functional.pad(h, (0, -d % 32)).view(n, -1, 32)
    top = pad.abs().amax(2, keepdim=True).clamp(min=2.0 ** -120)
    step = top / torch.frexp(top)[0] * 2.0 ** -7
    q = torch.clamp(torch.round(pad / step), -127, 127)
    return (q * step).view(n, -1)[:, :d]


def geglu_q8_plain(s):
    u = s["u"].detach().float()
    n, d = s["g"].shape
    a, b = u[:, :d], u[:, d:]
    z = GELU_C * (a + GELU_A * a * a * a)
    out = a / (1.0 + torch.exp(-2.0 * z)) * b
    a, b = quantised(a), quantised(b)
    sig = 1.0 / (1.0 + torch.exp(-2.0 * GELU_C * (a + GELU_A * a * a * a)))
    g = s["g"].float()
    da = g * b * (sig + a * sig * (1.0 - sig) * 2.0 * GELU_C * (1.0 + 3.0 * GELU_A * a * a))
    du = torch.cat([da, g * a * sig], 1)
    return out.to(s["u"].dtype), du.to(s["u"].dtype)


RUN = {("embedding", True): embedding_own, ("embedding", False): embedding_plain,
       ("cross_entropy", True): cross_entropy_own, ("cross_entropy", False): cross_entropy_plain,
       ("geglu_q8", True): geglu_q8_own, ("geglu_q8", False): geglu_q8_plain}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, d = case["n"], case["d"]
    es = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "geglu_q8":
        # forward: u read, out and the checkpoint (a byte a value, a byte a group of 32) written;
        # backward: the output's gradient and the checkpoint read, u's gradient written
        q8 = 2 * d + 2 * ((d + 31) // 32)
        return {"bytes": n * (2 * d * es + d * es + q8 + d * es + q8 + 2 * d * es), "flops": 0}
    v = case["vocab"]
    if case["op"] == "embedding":
        looked_up = n * 8 + min(n, v) * d * es + n * d * es
        return {"bytes": looked_up + (n * 8 + n * d * es + v * d * es if case["step"] else 0), "flops": 0}
    bytes_ = n * d * es + v * d * es + n * 8 + (n * 4 if case["reduction"] == "none" else 4)
    if case["step"]:
        bytes_ += n * d * es + v * d * es
    return {"bytes": bytes_, "flops": (6 if case["step"] else 2) * n * v * d}


# ---------------------------------------------------------------- the definitions in float64
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        table = s["table"].detach().double().requires_grad_(case["step"])
        out = torch.nn.functional.embedding(s["tokens"], table, padding_idx=case["padding"] if case["padding"] >= 0 else None)
        out = out * case["scale"]
        if not case["step"]:
            return out
        return out.detach(), torch.autograd.grad(out, table, s["g"].double())[0]
    if case["op"] == "cross_entropy":
        x = s["x"].detach().double().requires_grad_(case["step"])
        w = s["w"].detach().double().requires_grad_(case["step"])
        logits = torch.nn.functional.linear(x, w) * case["scale"]
        loss = torch.nn.functional.cross_entropy(logits, s["targets"], ignore_index=-100, reduction="none")
        if case["z_loss"]:
            loss = loss + case["z_loss"] * torch.logsumexp(logits, 1).square() * (s["targets"] != -100)
        up = None
        if case["reduction"] == "mean":
            loss = loss.sum() / max(1, int((s["targets"] != -100).sum()))
        elif case["reduction"] == "sum":
            loss = loss.sum()
        else:
            up = s["g"].double()
        if not case["step"]:
            return loss
        del logits
        dx, dw = torch.autograd.grad(loss, (x, w), up)
        return loss.detach(), dx, dw
    d = case["d"]
    u = s["u"].detach().double()

    def geglu(h):
        return torch.nn.functional.gelu(h[:, :d], approximate="tanh") * h[:, d:]

    kept = torch.empty_like(u)
    for half in (slice(0, d), slice(d, 2 * d)):
        for c0 in range(half.start, half.stop, 32):
            cols = slice(c0, min(c0 + 32, half.stop))
            m, e = torch.frexp(u[:, cols])   # u = m 2^e: in units of the largest leading power, 2^(top - 1)
            top = torch.where(m != 0, e, -119).amax(1, keepdim=True).clamp(min=-119)
            q = torch.round(torch.ldexp(m, e - top + 7)).clamp(-127, 127)
            kept[:, cols] = torch.ldexp(q, top - 7)
    kept.requires_grad_(True)
    return geglu(u), torch.autograd.grad(geglu(kept), kept, s["g"].double())[0]
