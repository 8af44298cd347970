"""Measured cases of what a training step does between its matrix products and of its products in 8 bits: the
residual's addition with the root-mean-square norm, forward and backward; the same with its output in 8 bits; the
projection that reads those 8 bits; and the AdamW step over all tensors of a model, its states in 32 or 8 bits.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds before the
call, run() makes one pass: with `own` false in elementary torch operations in fp32, with `own` true through this
library's public functions.  exact() gives a pass's values in float64.
"""
import importlib
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
LIBRARY = Path(__file__).resolve().parent.parent / "kernel-rsi_b200" / "library"
EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
GROUP = 256   # elements that share the two exponents of an 8-bit optimizer state
MASK = 0xFFFFFFFF


def library(name):
    """A module of the library (its folder goes on sys.path, as its users put it there)."""
    if str(LIBRARY) not in sys.path:
        sys.path.insert(0, str(LIBRARY))
    return importlib.import_module(name)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the junction of one short prompt's 16 tokens, without a gradient: latency
        {"name": "addnorm_16", "op": "add_rmsnorm", "n": 16, "d": 1152, "dtype": "bf16", "step": False},
        # a small fp32 model's step: odd rows, a width that is no multiple of a vector
        {"name": "addnorm_step_ragged", "op": "add_rmsnorm", "n": 5003, "d": 1149, "dtype": "f32", "step": True},
        # a junction of the block model's batch (32 sequences of 1024, d 1152), forward and backward
        {"name": "addnorm_step_32k", "op": "add_rmsnorm", "n": 32768, "d": 1152, "dtype": "bf16", "step": True},
        # the junction before a projection in 8 bits, odd rows and a row width of no whole 16 bytes, f16
        {"name": "addnorm8_ragged", "op": "add_rmsnorm_q8", "n": 1777, "d": 2740, "dtype": "f16"},
        # the same on the block model's batch
        {"name": "addnorm8_32k", "op": "add_rmsnorm_q8", "n": 32768, "d": 1152, "dtype": "bf16"},
        # the gate|value projection of 16 tokens: the weight's read is all there is
        {"name": "linear8_16", "op": "linear_q8", "n": 16, "d": 1152, "out": 9216, "dtype": "bf16"},
        # sizes that end inside every tile, fp32 out
        {"name": "linear8_ragged", "op": "linear_q8", "n": 2001, "d": 1000, "out": 2743, "dtype": "f32"},
        # the gate|value projection of the block model's batch
        {"name": "linear8_32k", "op": "linear_q8", "n": 32768, "d": 1152, "out": 9216, "dtype": "bf16"},
        # a one-layer fp32 model's update: launch and host
        {"name": "adamw_small", "op": "adamw", "layers": 1, "d": 72, "ff": 250, "vocab": 0, "dtype": "f32", "bits": 32,
         "master": False, "max_norm": 0.0},
        # the block model (28 layers), bf16 weights with fp32 masters, clipped by the global norm
        {"name": "adamw_28_layers", "op": "adamw", "layers": 28, "d": 1152, "ff": 4608, "vocab": 0, "dtype": "bf16",
         "bits": 32, "master": True, "max_norm": 1.0},
        # a two-layer f16 model with odd widths and states in 8 bits, clipped
        {"name": "adamw8_ragged", "op": "adamw", "layers": 2, "d": 501, "ff": 1333, "vocab": 10007, "dtype": "f16",
         "bits": 8, "master": True, "max_norm": 1.0},
        # the block model with its vocabulary's table, states in 8 bits and no masters: 10 bytes a weight
        {"name": "adamw8_28_layers", "op": "adamw", "layers": 28, "d": 1152, "ff": 4608, "vocab": 32768,
         "dtype": "bf16", "bits": 8, "master": False, "max_norm": 0.0},
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["add_rmsnorm", "add_rmsnorm_q8", "linear_q8", "adamw"])
    if op == "adamw":
        d = log_int(rng, 64, 1152)
        bits, dtype = rng.choice([32, 8]), rng.choice(["bf16", "bf16", "f16", "f32"])
        return {"op": op, "layers": log_int(rng, 1, 28), "d": d, "ff": log_int(rng, 2 * d, 4 * d),
                "vocab": rng.choice([0, log_int(rng, 1000, 32768)]), "dtype": dtype, "bits": bits,
                "master": dtype != "f32" and rng.random() < 0.5, "max_norm": rng.choice([0.0, 1.0])}
    n = log_int(rng, 1, 32768)
    if op == "linear_q8":
        d, out = log_int(rng, 64, 4608), log_int(rng, 64, 9216)
        return {"op": op, "n": min(n, 32768 * 1152 * 9216 // (d * out)), "d": d, "out": out,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    case = {"op": op, "n": n, "d": log_int(rng, 64, 4608), "dtype": rng.choice(["bf16", "f16", "f32"])}
    case["n"] = min(n, 32768 * 1152 * (1 if case["dtype"] == "f32" else 2) // (2 * case["d"]))
    if op == "add_rmsnorm":
        case["step"] = rng.random() < 0.75
    return case


def shapes(case):
    """A T5 encoder's tensors: four projections, gate, value, down, two norms and the bias table a layer; the
    vocabulary's table and the last norm."""
    d, ff = case["d"], case["ff"]
    layer = [(d, d)] * 4 + [(ff, d), (ff, d), (d, ff), (d,), (d,), (32, 16)]
    return layer * case["layers"] + ([(case["vocab"], d)] if case["vocab"] else []) + [(d,)]


def spans(case):
    """(offset, elements) of each tensor in one buffer; each begins at a multiple of GROUP."""
    at, found = 0, []
    for shape in shapes(case):
        n = math.prod(shape)
        found.append((at, n))
        at += -(-n // GROUP) * GROUP
    return found, at


def to8(x):
    """Rows in 8 bits and their scales, rows padded to whole 16 bytes as add_rmsnorm_q8() writes them."""
    top = x.abs().amax(1, keepdim=True)
    q = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=E4M3, device=x.device)[:, :x.shape[1]]
    q.copy_((x * (448.0 / top)).to(E4M3))
    return q, (top / 448.0)[:, 0].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "adamw":
        where, total = spans(case)
        index = torch.zeros(total, dtype=torch.bool, device="cuda")
        for at, n in where:
            index[at:at + n] = True

        # gradients of very different sizes from group to group, a tenth of them zero
        def values(std, spread, zeros=0.0):
            v = normal(total) * std
            v *= torch.exp(spread * normal(total // GROUP)).repeat_interleave(GROUP)
            if zeros:
                v *= torch.rand(total, generator=g, device="cuda") >= zeros
            return v.mul_(index)

        p = values(0.02, 0.2)
        state = {"case": case, "grad": values(1e-4, 1.0, 0.1).to(dt), "step": torch.full((), 100, device="cuda")}
        state["p"] = p.to(dt)
        state["master"] = p if case["master"] else None
        m, v = values(3e-5, 1.0), values(1e-4, 1.0).square_()
        if case["bits"] == 8:
            state["m"], state["v"], state["exponents"] = encode(m, v, torch.zeros_like(m, dtype=torch.int32))
        else:
            state["m"], state["v"] = m, v
        kinds = ("p", "grad", "m", "v") + (("master",) if case["master"] else ())
        state["lists"] = {k: [state[k][at:at + n] for at, n in where] for k in kinds}
        if case["bits"] == 8:
            state["lists"]["exponents"] = [state["exponents"][at // GROUP:(at + n + GROUP - 1) // GROUP]
                                           for at, n in where]
        state["starts"] = torch.tensor([at for at, _ in where], device="cuda").repeat_interleave(
            torch.tensor([-(-n // GROUP) for _, n in where], device="cuda"))   # of each group's tensor
        return state

    n, d = case["n"], case["d"]
    if case["op"] == "linear_q8":
        q, scale = to8(normal(n, d) * torch.exp(0.5 * normal(n, 1)))
        wq, wscale = to8(normal(case["out"], d) * d ** -0.5)
        return {"case": case, "q": q, "scale": scale, "wq": wq, "wscale": wscale}

    # a residual stream of rows at scales of their own with a few columns far larger, and a sublayer's output
    res = normal(n, d) * torch.exp(0.5 * normal(n, 1)) * torch.exp(0.7 * normal(1, d))
    s = {"case": case, "x": normal(n, d).to(dt), "res": res.to(dt), "w": (1 + 0.1 * normal(d)).to(dt)}
    if case.get("step"):
        s["gy"], s["gz"] = normal(n, d).to(dt), normal(n, d).to(dt)
        for k in ("x", "res", "w"):
            s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    return RUN[state["case"]["op"], bool(own)](state)


def add_rmsnorm_own(s):
    y, z = library("add_rmsnorm").add_rmsnorm(s["x"], s["res"], s["w"], EPS)
    if not s["case"]["step"]:
        return y, z
    return (y.detach(), z.detach(), *torch.autograd.grad((y, z), (s["x"], s["res"], s["w"]), (s["gy"], s["gz"])))


def add_rmsnorm_plain(s):
    x, res, w = (s[k].detach() for k in ("x", "res", "w"))
    z = (x.float() + res.float()).to(x.dtype)
    z32, w32 = z.float(), w.float()
    r = 1.0 / torch.sqrt(z32.square().mean(1, keepdim=True) + EPS)
    n = z32 * r
    y = (n * w32).to(x.dtype)
    if not s["case"]["step"]:
        return y, z
    gy = s["gy"].float()
    dw = (gy * n).sum(0)
    gw = gy * w32
    dz = r * (gw - n * (gw * n).mean(1, keepdim=True)) + s["gz"].float()
    dz = dz.to(x.dtype)
    return y, z, dz, dz, dw.to(w.dtype)


def add_rmsnorm_q8_own(s):
    return library("add_rmsnorm").add_rmsnorm_q8(s["x"], s["res"], s["w"], EPS)


def add_rmsnorm_q8_plain(s):
    x, res, w = s["x"], s["res"], s["w"]
    z = (x.float() + res.float()).to(x.dtype)
    z32 = z.float()
    r = 1.0 / torch.sqrt(z32.square().mean(1, keepdim=True) + EPS)
    t = z32 * w.float()
    top = t.abs().amax(1, keepdim=True)
    q = (t * (448.0 / top)).to(E4M3)
    return q, (top * r / 448.0)[:, 0], z


def linear_q8_own(s):
    return library("linear_q8").linear_q8(s["q"], s["scale"], s["wq"], s["wscale"], DTYPES[s["case"]["dtype"]])


def linear_q8_plain(s):
    out = s["q"].float() @ s["wq"].float().t()
    return out.mul_(s["scale"][:, None]).mul_(s["wscale"]).to(DTYPES[s["case"]["dtype"]])


def outputs(s, norm):
    kinds = ("p", "master", "m", "v", "exponents", "step")
    return {**{k: s[k] for k in kinds if s.get(k) is not None}, **({} if norm is None else {"norm": norm})}


def adamw_own(s):
    c, lists = s["case"], s["lists"]
    norm = library("adamw").adamw_step(
        lists["p"], lists["grad"], lists["m"], lists["v"], s["step"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
        weight_decay=DECAY, max_norm=c["max_norm"], masters=lists.get("master"), exponents=lists.get("exponents"))
    return outputs(s, norm)


def dither(starts, total, step):
    """16 bits for each element, from its place in its tensor and the step."""
    i = torch.arange(total, device=starts.device).view(-1, GROUP)
    i = (i - starts[:, None]).view(-1)
    h = ((i >> 1) * 0x9E3779B1 + step * 0x632BE5AB) & MASK
    h = ((h ^ (h >> 16)) * 0x21F0AAAD) & MASK
    h = ((h ^ (h >> 15)) * 0x735A2D97) & MASK
    h = h ^ (h >> 15)
    return ((h >> (16 * (i & 1))) & 0xFFFF).int()


def exponent(top):
    """The exponent field of a positive fp32."""
    return top.view(torch.int32) >> 23


def power(byte):
    return (byte.int() << 23).view(torch.float32)


def encode(m, v, random16):
    """The first moments and the second ones' square roots in 8 bits: e4m3 at a power of two for each group, its
    largest magnitude in [128, 256); the first to nearest, the roots up or down by the dither, never down to 0."""
    m, v = m.view(-1, GROUP), v.view(-1, GROUP)
    em = (exponent(m.abs().amax(1)) - 7).clamp(1, 254)
    er = (((exponent(v.amax(1)) - 127) >> 1) + 120).clamp(1, 254)
    m8 = (m * power(254 - em)[:, None]).to(E4M3)
    r = torch.sqrt(v) * power(254 - er)[:, None]
    lift = torch.where(r < 2.0 ** -6, 2.0 ** -6, 0.0)
    up = ((r + lift).view(torch.int32) + (random16.view(-1, GROUP) << 4)) & ~0xFFFFF
    r8 = torch.where(r > 0, (up.view(torch.float32) - lift).clamp(min=2.0 ** -9), 0.0).to(E4M3)
    return m8.view(-1), r8.view(-1), torch.stack([em, er], 1).to(torch.uint8)


def adamw_plain(s):
    c, grad = s["case"], s["grad"].float()
    s["step"] += 1
    norm = None
    if c["max_norm"]:
        norm = torch.sqrt(grad.square().sum(dtype=torch.float64)).float()
        grad = grad * torch.clamp(c["max_norm"] / (norm + 1e-6), max=1.0)
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        scales = power(s["exponents"])
        m = (m.float().view(-1, GROUP) * scales[:, :1]).view(-1)
        v = (v.float().view(-1, GROUP) * scales[:, 1:]).view(-1).square_()
    m.mul_(BETA1).add_(grad * (1 - BETA1))
    v.mul_(BETA2).add_(grad.square().mul_(1 - BETA2))
    if c["bits"] == 8:
        m8, r8, exponents = encode(m, v, dither(s["starts"], m.numel(), s["step"]))
        s["m"].copy_(m8), s["v"].copy_(r8), s["exponents"].copy_(exponents)
    t = s["step"].double()
    rate = (LR / (1 - BETA1 ** t)).float()
    root = torch.sqrt(v).div_(torch.sqrt(1 - BETA2 ** t).float()).add_(ADAM_EPS)
    p = s["master"] if c["master"] else s["p"].float()
    p.mul_(1 - LR * DECAY).sub_(m.div(root).mul_(rate))
    s["p"].copy_(p)
    return outputs(s, norm)


RUN = {("add_rmsnorm", True): add_rmsnorm_own, ("add_rmsnorm", False): add_rmsnorm_plain,
       ("add_rmsnorm_q8", True): add_rmsnorm_q8_own, ("add_rmsnorm_q8", False): add_rmsnorm_q8_plain,
       ("linear_q8", True): linear_q8_own, ("linear_q8", False): linear_q8_plain,
       ("adamw", True): adamw_own, ("adamw", False): adamw_plain}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    es = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in shapes(case))
        # read and written: weight, both states (two exponents a group in 8 bits) and the master; the gradient read,
        # a second time where its norm has to be known first; a weight with a master is written only
        state = 2 * (2 + 2 / GROUP) if case["bits"] == 8 else 2 * 8
        weight = es + 8 if case["master"] else 2 * es
        return {"bytes": n * (weight + state + es * (2 if case["max_norm"] else 1)), "flops": 0}
    n, d = case["n"], case["d"]
    if case["op"] == "linear_q8":
        out = case["out"]
        return {"bytes": n * (d + 4) + out * (d + 4) + n * out * es, "flops": 2 * n * d * out}
    if case["op"] == "add_rmsnorm_q8":
        return {"bytes": n * d * (3 * es + 1) + n * 4 + d * es, "flops": 0}
    # x and the residual read, their sum and the norm written; backward: the sum and both gradients read, the
    # gradients of x and w written
    return {"bytes": n * d * es * (8 if case["step"] else 4) + (3 if case["step"] else 1) * d * es, "flops": 0}


# ---------------------------------------------------------------- the definitions in float64
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return exact_adamw(s)
    if case["op"] == "linear_q8":
        out = torch.empty(case["n"], case["out"], dtype=torch.float64, device="cuda")
        w = s["wq"].double() * s["wscale"].double()[:, None]
        for i in range(0, case["n"], 4096):
            out[i:i + 4096] = torch.nn.functional.linear(s["q"][i:i + 4096].double() * s["scale"][i:i + 4096, None], w)
        return out
    dt = s["x"].dtype
    z = (s["x"].detach().double() + s["res"].detach().double()).to(dt).double().requires_grad_(True)
    w = s["w"].detach().double().requires_grad_(True)
    y = torch.nn.functional.rms_norm(z, (case["d"],), w, eps=EPS)
    if case["op"] == "add_rmsnorm":
        if not case["step"]:
            return y.detach(), z.detach()
        dz, dw = torch.autograd.grad(y, (z, w), s["gy"].double())
        dz = dz + s["gz"].double()
        return y.detach(), z.detach(), dz, dz, dw
    y = y.detach()
    scale = y.abs().amax(1) / 448
    a, e = torch.frexp(y / scale[:, None])      # e4m3: four leading bits, down to 2^-9
    e = e.clamp(min=-5)
    q = torch.ldexp(torch.round(torch.ldexp(y / scale[:, None], 4 - e)), e - 4)
    return q, scale, z.detach()


def exact_adamw(s):
    c = s["case"]
    g = s["grad"].double()
    norm = g.norm()
    if c["max_norm"]:
        g = g * min(1.0, c["max_norm"] / (norm.item() + 1e-6))
    t = int(s["step"]) + 1
    m, v = s["m"].double(), s["v"].double()
    if c["bits"] == 8:
        scales = torch.exp2(s["exponents"].double() - 127).repeat_interleave(GROUP, 0)
        m, v = m * scales[:, 0], (v * scales[:, 1]) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = s["master"].double() if c["master"] else s["p"].double()
    p = p * (1 - LR * DECAY)
    p -= LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    out = {"p": p, "m": m, "v": v, "step": None}
    if c["master"]:
        out["master"] = p
    if c["max_norm"]:
        out["norm"] = norm
    if c["bits"] == 8:
        tops = m.view(-1, GROUP).abs().amax(1), v.view(-1, GROUP).amax(1).sqrt()
        em, er = (torch.frexp(top)[1].sub(8).clamp(min=-126).repeat_interleave(GROUP) for top in tops)
        del tops
        a = torch.ldexp(m, -em)
        e = torch.frexp(a)[1].clamp(min=-5)
        out["m"] = torch.ldexp(torch.round(torch.ldexp(a, 4 - e)), e - 4)
        del a, m, g
        r = torch.ldexp(v.sqrt(), -er)
        e = torch.frexp(r)[1].clamp(min=-5)
        low = torch.floor(torch.ldexp(r, 4 - e) + dither(s["starts"], r.numel(), t).double() * 2.0 ** -16)
        out["v"] = torch.where(r > 0, torch.ldexp(low, e - 4).clamp(min=2.0 ** -9), 0.0)
        out["exponents"] = None
    return out
