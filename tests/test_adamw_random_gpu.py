"""8-bit states whose first moments are rounded at random too: the codes bit for bit against the rule restated in torch,
and runs of steps beside fp32 states, which is what the rounding is for."""
import copy
import math
import warnings

import pytest
import torch

import adamw
from adamw import GROUP, AdamW, adamw_step, dequantise, new_state

pytestmark = pytest.mark.gpu
dev = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3 = torch.float8_e4m3fn
B1, B2 = 0.9, 0.999
HYPER = dict(lr=1e-2, betas=(B1, B2), eps=1e-8, weight_decay=0.1, rounding="random")
SIZES = [1, 7, 255, 256, 257, 0, 8191, 8192, 8193, 40000, 3]
KINDS = [(F32, F32, False), (BF16, BF16, False), (BF16, BF16, True), (BF16, F32, False), (BF16, F32, True),
         (F16, F16, False), (F16, F16, True), (F16, F32, False), (F16, F32, True)]
BETAS = [(0.9, 0.999), (0.9, 0.95), (0.95, 0.95), (0.97, 0.999), (0.99, 0.999)]


def count(t=0):
    return torch.full((), t, dtype=torch.int64, device=dev)


def raw(t):
    return t.contiguous().reshape(-1).view(torch.uint8)


# ---------------------------------------------------------------- the rule
def words(n, step):
    """For each element 16 bits that round sqrt(v) and 16 that round m."""
    i, mask = torch.arange(n, device=dev), 0xFFFFFFFF
    h = ((i >> 1) * 0x9E3779B1 + step * 0x632BE5AB) & mask
    h = ((h ^ (h >> 16)) * 0x21F0AAAD) & mask
    h = ((h ^ (h >> 15)) * 0x735A2D97) & mask
    h = h ^ (h >> 15)
    k = (h * 0x2C1B3C6D) & mask
    k = k ^ (k >> 16)
    return [((x >> (16 * (i & 1))) & 0xFFFF).int() for x in (h, k)]


def power(byte):
    return (byte.int() << 23).view(F32)


def up_or_down(x, random16):
    """Magnitudes in [0, 256] to a multiple of their code's last bit."""
    lift = torch.where(x < 2.0 ** -6, 2.0 ** -6, 0.0)
    return (((x + lift).view(torch.int32) + (random16 << 4)) & ~0xFFFFF).view(F32) - lift


def rule(g, m8, r8, exponents, clip, step):
    n = g.numel()
    pad = lambda x: torch.nn.functional.pad(x, (0, -n % GROUP)).view(-1, GROUP)  # noqa: E731
    s, (for_r, for_m) = power(exponents), map(pad, words(n, step))
    m, r = pad(m8.float()) * s[:, :1], pad(r8.float()) * s[:, 1:]
    g = pad(g.float() * clip)
    m = m * B1 + g * (1 - B1)
    v = (r * r) * B2 + (g * g) * (1 - B2)
    em = ((m.abs().amax(1).view(torch.int32) >> 23) - 7).clamp(1, 254)
    er = (((v.amax(1).view(torch.int32) >> 23) - 127) >> 1) + 120
    x, r = m * power(254 - em)[:, None], v.sqrt() * power(254 - er)[:, None]
    m = torch.copysign(up_or_down(x.abs(), for_m), x)
    r = torch.where(r > 0, up_or_down(r, for_r).clamp(min=2.0 ** -9), 0.0)
    flat = lambda x: x.to(E4M3).view(-1)[:n]  # noqa: E731
    return flat(m), flat(r), torch.stack([em, er], 1).to(torch.uint8)


def make(sizes, pt, gt=None, master=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    lists = {k: [] for k in ("p", "g", "m", "v", "master", "exponents")}
    for n in sizes:
        rand = lambda s=1.0: (torch.randn(n, generator=g) * s).to(dev)  # noqa: E731
        p = rand()
        lists["p"].append(p.to(pt))
        # gradients over many binades, a tenth of them zero
        lists["g"].append((rand(0.1) * torch.exp2(4 * rand()) * (rand() > -1.3)).to(gt or pt))
        for k, x in zip(("m", "v", "exponents"), new_state(p, 8)):
            lists[k].append(x)
        lists["master"].append(p.clone() if master and pt != F32 else torch.zeros(0, device=dev))
    return lists


def call(l, step, **kw):
    return adamw_step(l["p"], l["g"], l["m"], l["v"], step, masters=l["master"], exponents=l["exponents"],
                      **{**HYPER, **kw})


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("pt,gt,master", KINDS)
def test_codes_follow_the_rule(pt, gt, master, max_norm):
    """Bit for bit over several steps; the parameter moves by the moments before they are rounded, as with any rounding:
    its values are those of the nearest codes' call on the same states."""
    l = make(SIZES, pt, gt, master=master)
    step = count()
    for t in (1, 2, 3, 4):
        old = copy.deepcopy(l)
        norm = call(l, step, max_norm=max_norm)
        clip = torch.clamp(max_norm / (norm + 1e-6), max=1.0) if max_norm else 1.0
        for i in range(len(SIZES)):
            want = rule(l["g"][i], old["m"][i], old["v"][i], old["exponents"][i], clip, t)
            for a, b in zip((l["m"][i], l["v"][i], l["exponents"][i]), want):
                assert torch.equal(raw(a), raw(b))
        call(old, count(t - 1), max_norm=max_norm, rounding="nearest")
        for k in ("p", "master", "v", "exponents"):
            assert all(torch.equal(raw(a), raw(b)) for a, b in zip(l[k], old[k]))
        for x in l["g"]:
            x.mul_(-0.3)
            x[256:512] = 0


@pytest.mark.parametrize("pt", [F32, BF16])
def test_codes_on_borders(pt):
    """Every pair of a code of m and a short gradient: sums on codes, between codes, in the subnormal ones, zero and of
    either sign."""
    n = 1 << 20
    l = make([n], pt)
    g = torch.Generator().manual_seed(5)
    codes = torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8)
    codes[(codes & 0x7F) >= 0x78] = 0   # (up to 240, as the group's largest is)
    l["m"][0].copy_(codes.view(E4M3))
    l["v"][0].copy_(torch.randint(1, 41, (n,), generator=g).to(E4M3))
    l["exponents"][0].copy_(torch.randint(100, 104, (n // GROUP, 2), generator=g))
    few = torch.randint(-160, 161, (n,), generator=g) * 2.0 ** torch.randint(-40, -25, (n,), generator=g)
    l["g"][0].copy_(few * (torch.rand(n, generator=g) < 0.7))
    want = rule(l["g"][0], l["m"][0], l["v"][0], l["exponents"][0], 1.0, 1)
    call(l, count())
    for a, b in zip((l["m"][0], l["v"][0], l["exponents"][0]), want):
        assert (raw(a) != raw(b)).sum().item() == 0


def test_one_step_is_right_on_average():
    """Each element's code is one of the two beside its value, and the errors' mean over N elements is within 6 standard
    deviations, half a code (at most 2^-4 of a value, 2^-10 of the unit) over N^0.5 each."""
    n = 1 << 18
    l = make([n], F32)
    l["g"][0].copy_(torch.exp2(-14 * torch.rand(n, generator=torch.Generator().manual_seed(1))))
    call(l, count())
    m, _ = dequantise(l["m"][0], l["v"][0], l["exponents"][0])
    unit = power(l["exponents"][0][:, 0]).double().repeat_interleave(GROUP)
    want = (1 - B1) * l["g"][0].double()
    off, one = m.double() - want, torch.maximum(want * 2.0 ** -3, unit * 2.0 ** -9)
    assert (off.abs() <= one * (1 + 1e-6)).all()
    assert abs((off / one).mean().item()) <= 6 * 0.5 / n ** 0.5


# ---------------------------------------------------------------- runs of steps
def run(grads, steps, betas, bits):
    """A parameter's travel in units of lr under grads(t), from 0 in fp32, and its optimizer."""
    p = torch.zeros(1 << 14, device=dev, requires_grad=True)
    opt = AdamW([p], lr=1.0, betas=betas, eps=1e-12, weight_decay=0.0, bits=bits)
    for t in range(1, steps + 1):
        p.grad = grads(t)
        opt.step()
    return p.detach().double(), opt.state[p]


@pytest.mark.parametrize("betas", BETAS)
def test_a_constant_gradient(betas):
    """m's mean is the gradient (the recursion is linear and the rounding right on average): the mean over 16384 elements
    of m / g, each within a code of 1 (2^-3) once settled, or within b1^t + 2^-4 / (1 - b1^2)^0.5 (0.5 for 0.99) on its way
    there, is within 6 x 0.5 / 128 of 1.  The travel in 1000 steps is lr a step over r / g: two neighbouring codes of r make
    the mean of its inverse 2^-9 too large, the first steps' rounding (5% rms, kept for 1 / (1 - b2) steps) as much
    again and 2^-3 / 128 at random: 2%."""
    g = torch.randn(1 << 14, generator=torch.Generator().manual_seed(0)).abs().mul(1e-3).add(1e-4).to(dev)
    want, _ = run(lambda t: g, 1000, betas, 32)
    got, state = run(lambda t: g, 1000, betas, 8)
    m, _ = dequantise(state["exp_avg"], state["exp_avg_sq"], state["exponents"])
    settled = 1 - betas[0] ** 1000
    assert abs((m.double() / g).mean().item() / settled - 1) <= 6 * 0.5 / 128
    assert abs((got / want).mean().item() - 1) <= 0.02


@pytest.mark.parametrize("size", [0.01, 1.0])
@pytest.mark.parametrize("betas", BETAS)
def test_a_group_of_which_half_goes_idle(betas, size):
    """Gradients at random for one half of each group; the other half has some, `size` as large, for 20 steps and none for
    1500 more.  Its m goes to zero, and its weights stop where fp32 states leave them.  The root mean square of their
    travel is then off by the noise of m (each step's at most 2^-4 of m, 2^-4 / (1 - b1^2)^0.5 of the travel: 0.44 for 0.99,
    which as a root of squares makes 1.09) and of r (jumps of a code, whose inverses' mean is up to a tenth larger while m
    decays): a quarter."""
    gen = torch.Generator().manual_seed(1)
    noise = [torch.randn(1 << 14, generator=gen).to(dev) for _ in range(64)]
    idle = torch.arange(1 << 14, device=dev) % GROUP >= GROUP // 2

    def grads(t):
        g = noise[t % 64].clone()
        g[idle] *= size if t <= 20 else 0.0
        return g

    rms = lambda p: p[idle].square().mean().sqrt().item()  # noqa: E731
    want, got = (run(grads, 1520, betas, bits) for bits in (32, 8))
    assert rms(want[0]) / 1.25 <= rms(got[0]) <= 1.25 * rms(want[0])
    # after 1500 steps an element still has a code with the probability b1^1500 of its last value's, at most 2^17 least codes
    m = got[1]["exp_avg"].float()[idle]
    assert (m != 0).float().mean().item() <= 0.001 + 2 ** 17 * betas[0] ** 1500


# ---------------------------------------------------------------- calls
def test_addresses_order_and_graphs_do_not_show():
    """The same bits for tensors off 16 bytes, for gradients in another order, through the dispatcher, in a graph that is
    replayed, and among other tensors."""
    base = make([3000], BF16, master=True)
    want = copy.deepcopy(base)
    call(want, count()), call(want, count(1))

    def same(l):
        return all(torch.equal(raw(a), raw(b)) for k in ("p", "m", "v", "exponents", "master") for a, b in zip(l[k], want[k]))

    moved = copy.deepcopy(base)
    for k in ("p", "g", "m", "v", "master"):
        x = moved[k][0]
        room = torch.zeros(x.numel() + 3, dtype=x.dtype, device=dev)
        room[3:].copy_(x)
        moved[k] = [room[3:]]
    call(moved, count()), call(moved, count(1))
    assert same(moved)
    two = copy.deepcopy(base)
    for k in ("p", "g", "m", "v", "master"):
        two[k] = [two[k][0].view(50, 60)]
    two["g"] = [two["g"][0].t().contiguous().t()]
    call(two, count()), call(two, count(1))
    assert same(two)
    boxed = copy.deepcopy(base)
    for t in (0, 1):
        torch.ops.krsi.adamw_step(boxed["p"], boxed["g"], boxed["m"], boxed["v"], boxed["master"], boxed["exponents"],
                                  count(t), None, 1e-2, B1, B2, 1e-8, 0.1, 0.0, True)
    assert same(boxed)
    compiled = copy.deepcopy(base)
    fn = torch.compile(lambda s: call(compiled, s))
    fn(count()), fn(count(1))
    assert same(compiled)
    many = copy.deepcopy(base)
    others = make([300] * 30, F32, seed=3)
    every = {k: others[k][:7] + many[k] + others[k][7:] for k in many}
    step = count()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call(every, step)
    graph.replay(), graph.replay()
    assert step.item() == 2 and same(many)


def test_not_finite_values_mark_their_group():
    for bad in (float("nan"), float("inf"), float("-inf")):
        l = make([600], F32)
        l["g"][0][300] = bad
        call(l, count())
        m, v = dequantise(l["m"][0], l["v"][0], l["exponents"][0])
        assert torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
        assert torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all()


def test_the_default_says_what_it_is(monkeypatch):
    monkeypatch.setattr(adamw, "_warned", False)
    plain, named = make([600], F32), make([600], F32)
    no_name = {k: v for k, v in HYPER.items() if k != "rounding"}
    with pytest.warns(UserWarning, match="rounding"):
        adamw_step(plain["p"], plain["g"], plain["m"], plain["v"], count(), exponents=plain["exponents"], **no_name)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        adamw_step(plain["p"], plain["g"], plain["m"], plain["v"], count(1), exponents=plain["exponents"], **no_name)
        monkeypatch.setattr(adamw, "_warned", False)
        call(named, count(), rounding="nearest"), call(named, count(1), rounding="nearest")
        p = torch.zeros(5000, device=dev, requires_grad=True)
        p.grad = torch.ones_like(p)
        AdamW([p], bits=8).step()
    assert all(torch.equal(raw(a), raw(b)) for k in ("p", "m", "v") for a, b in zip(plain[k], named[k]))
    with pytest.raises(ValueError, match="rounding"):
        call(named, count(), rounding="up")
