"""adamw_step and the AdamW optimizer against the update's definition in float64.

Tolerances: fp32 operations are off by 2^-24 of their result each.  The moments take four; the update's quotient
eight and what the moments' errors give it; the parameter two more and its type's rounding.  8-bit states are held
to their rule bit for bit: it is made of IEEE operations in a fixed order, restated here in torch."""
import copy

import pytest
import torch

import _ext
from adamw import GROUP, AdamW, adamw_step, dequantise, new_state

pytestmark = pytest.mark.gpu
dev = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 0.1
HYPER = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)


def count(t=0):
    return torch.full((), t, dtype=torch.int64, device=dev)


def make(sizes, pt, gt=None, bits=32, master=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    lists = {k: [] for k in ("p", "g", "m", "v", "master", "exponents")}
    for n in sizes:
        rand = lambda s=1.0: (torch.randn(n, generator=g) * s).to(dev)  # noqa: E731
        p = rand()
        lists["p"].append(p.to(pt))
        lists["g"].append((rand(0.1) * (rand() > -1.0)).to(gt or pt))
        m, v, e = new_state(p, bits)
        if bits == 32:
            m.copy_(rand(0.05)), v.copy_(rand(0.1).square())
        lists["m"].append(m), lists["v"].append(v), lists["exponents"].append(e)
        lists["master"].append(p.clone() if master and pt != F32 else torch.zeros(0, device=dev))
    return lists


def call(l, step, **kw):
    return adamw_step(l["p"], l["g"], l["m"], l["v"], step, masters=l["master"], exponents=l["exponents"],
                      **{**HYPER, **kw})


def check(before, after, t, clip=1.0):
    """One tensor after a step from (p or master, g, m, v): float64, elementwise."""
    p, g, m, v = (x.double() for x in before)
    p1, m1, v1 = after
    e = 2 ** -24
    g = g * clip
    m64, v64 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    dm = 8 * e * (B1 * m.abs() + (1 - B1) * g.abs())
    assert ((m1.double() - m64).abs() <= dm).all()
    assert ((v1.double() - v64).abs() <= 8 * e * v64).all()
    root = (v64 / (1 - B2 ** t)).sqrt() + EPS
    move = LR / (1 - B1 ** t) * m64 / root
    p64 = p * (1 - LR * WD) - move
    tol = 16 * e * move.abs() + LR / (1 - B1 ** t) * dm / root + 3 * e * p.abs()
    half = torch.finfo(p1.dtype).eps / 2
    low = torch.finfo(p1.dtype).tiny * half   # half a step of the subnormals: f16 has them from 2^-14 (2^-25 off)
    assert ((p1.double() - p64).abs() <= half * p64.abs() + low + tol * (1 + half)).all()


SIZES = [1, 7, 255, 256, 257, 0, 8191, 8192, 8193, 40000, 3]
KINDS = [(F32, F32, False), (BF16, BF16, False), (BF16, BF16, True), (BF16, F32, False), (BF16, F32, True),
         (F16, F16, False), (F16, F16, True), (F16, F32, False), (F16, F32, True)]


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("pt,gt,master", KINDS)
def test_step_against_float64(pt, gt, master, max_norm):
    l = make(SIZES, pt, gt, master=master)
    before = [[x.clone() for x in s] for s in zip(l["master"] if master else l["p"], l["g"], l["m"], l["v"])]
    step = count(4)
    norm = call(l, step, max_norm=max_norm)
    assert step.item() == 5
    clip = 1.0
    if max_norm:
        want = torch.cat(l["g"]).double().norm()
        assert abs(norm.double() - want) <= 2 ** -23 * want
        clip = min(1.0, max_norm / (want.item() + 1e-6))
        assert clip < 1
    else:
        assert norm is None
    for i, b in enumerate(before):
        check(b, ((l["master"] if master else l["p"])[i], l["m"][i], l["v"][i]), 5, clip)
        if master:
            assert torch.equal(l["p"][i], l["master"][i].to(pt))


# ---------------------------------------------------------------- 8-bit states
def dither(n, step):
    i, mask = torch.arange(n, device=dev), 0xFFFFFFFF
    h = ((i >> 1) * 0x9E3779B1 + step * 0x632BE5AB) & mask
    h = ((h ^ (h >> 16)) * 0x21F0AAAD) & mask
    h = ((h ^ (h >> 15)) * 0x735A2D97) & mask
    h = h ^ (h >> 15)
    return (h >> (16 * (i & 1))) & 0xFFFF


def power(byte):
    return (byte.int() << 23).view(F32)


def rule(g, m8, r8, exponents, clip, step):
    """(m8, r8, exponents) after a step, in fp32 operations."""
    n = g.numel()
    pad = lambda x: torch.nn.functional.pad(x, (0, -n % GROUP)).view(-1, GROUP)  # noqa: E731
    s = power(exponents)
    m, r = pad(m8.float()) * s[:, :1], pad(r8.float()) * s[:, 1:]
    g = pad(g.float() * clip)
    m = m * B1 + g * (1 - B1)
    v = (r * r) * B2 + (g * g) * (1 - B2)
    em = ((m.abs().amax(1).view(torch.int32) >> 23) - 7).clamp(1, 254)
    er = (((v.amax(1).view(torch.int32) >> 23) - 127) >> 1) + 120
    r = v.sqrt() * power(254 - er)[:, None]
    lift = torch.where(r < 2.0 ** -6, 2.0 ** -6, 0.0)
    up = ((r + lift).view(torch.int32) + (pad(dither(n, step).int()) << 4)) & ~0xFFFFF
    r = torch.where(r > 0, (up.view(F32) - lift).clamp(min=2.0 ** -9), 0.0)
    flat = lambda x: x.to(torch.float8_e4m3fn).view(-1)[:n]  # noqa: E731
    return flat(m * power(254 - em)[:, None]), flat(r), torch.stack([em, er], 1).to(torch.uint8)


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("pt,gt,master", KINDS)
def test_8_bit_states_follow_their_rule(pt, gt, master, max_norm):
    l = make(SIZES, pt, gt, bits=8, master=master)
    step = count()
    for t in (1, 2, 3):
        before = [[x.clone() for x in s] for s in zip(l["master"] if master else l["p"], l["g"])]
        moments = [dequantise(m, v, e) for m, v, e in zip(l["m"], l["v"], l["exponents"])]
        want = None
        old = [[x.clone() for x in s] for s in zip(l["m"], l["v"], l["exponents"])]
        norm = call(l, step, max_norm=max_norm)
        clip = torch.clamp(max_norm / (norm + 1e-6), max=1.0) if max_norm else 1.0
        for i, n in enumerate(SIZES):
            want = rule(l["g"][i], *old[i], clip, t)
            for a, b in zip((l["m"][i], l["v"][i], l["exponents"][i]), want):
                assert torch.equal(bits(a), bits(b))
            # the parameter moves by the moments before they are rounded
            p, g = before[i]
            g = g.float() * clip
            m1 = B1 * moments[i][0] + (1 - B1) * g
            v1 = B2 * moments[i][1] + (1 - B2) * g * g
            check((p, g, *moments[i]), ((l["master"] if master else l["p"])[i], m1, v1), t)
        for x in l["g"]:   # gradients of another size the next time, some groups all zero
            x.mul_(0.3)
            x[256:512] = 0


@pytest.mark.parametrize("pt", [F32, BF16, F16])
def test_8_bit_codes_on_borders(pt):
    """0.9 m + 0.1 g of short m and g often lies on the border between two codes, where the last bit of the sum decides:
    the products are rounded before they are added."""
    n = 1 << 20
    l = make([n], pt, bits=8)
    g = torch.Generator().manual_seed(5)
    m, r = torch.randint(-40, 41, (n,), generator=g) * 4.0, torch.randint(1, 41, (n,), generator=g) * 4.0
    l["m"][0].copy_(m.to(torch.float8_e4m3fn)), l["v"][0].copy_(r.to(torch.float8_e4m3fn))
    l["exponents"][0].copy_(torch.randint(100, 104, (n // GROUP, 2), generator=g))
    l["g"][0].copy_(torch.randint(-160, 161, (n,), generator=g) * 2.0 ** -26)
    want = rule(l["g"][0], l["m"][0], l["v"][0], l["exponents"][0], 1.0, 1)
    call(l, count())
    for a, b in zip((l["m"][0], l["v"][0], l["exponents"][0]), want):
        assert (bits(a) != bits(b)).sum().item() == 0


def test_8_bit_values():
    """What the codes stand for: m within half a code of its value, the root within one code, positive ones not 0."""
    l = make([100000], F32, bits=8)
    l["g"][0].mul_(torch.exp2(torch.randint(-12, 3, (100000,)).to(dev).float()))
    g = l["g"][0].double()
    call(l, count())
    m, v = dequantise(l["m"][0], l["v"][0], l["exponents"][0])
    top = torch.exp2(l["exponents"][0].double() - 127).repeat_interleave(GROUP, 0)[:100000]
    m64, r64 = (1 - B1) * g, ((1 - B2) * g * g).sqrt()
    assert ((m.double() - m64).abs() <= 2 ** -4 * 1.001 * m64.abs() + 2 ** -10 * top[:, 0]).all()
    assert ((v.double().sqrt() - r64).abs() <= 2 ** -3 * 1.001 * r64 + 2 ** -9 * top[:, 1]).all()
    assert (v[g != 0] > 0).all() and (v[g == 0] == 0).all()


def test_the_rounding_is_right_on_average():
    """Without gradients r = sqrt(v) shrinks by sqrt(b2) a step, far less than a code.  Each step's rounding is at
    most a code (2^-3 of r) with variance a quarter of its square; over N elements and T steps the mean of r
    is within 6 standard deviations, 6 sqrt(T / 4) 2^-3 / sqrt(N), of r0 b2^(T / 2)."""
    N, T = 1 << 18, 300
    l = make([N], F32, bits=8)
    l["g"][0].fill_(1.0)
    step = count()
    call(l, step)
    r0 = dequantise(l["m"][0], l["v"][0], l["exponents"][0])[1].sqrt().double().mean().item()
    l["g"][0].zero_()
    for _ in range(T):
        call(l, step)
    r = dequantise(l["m"][0], l["v"][0], l["exponents"][0])[1].sqrt().double().mean().item()
    assert abs(r / r0 - B2 ** (T / 2)) <= 6 * (T / 4) ** 0.5 * 2 ** -3 / N ** 0.5
    assert abs(B2 ** (T / 2) - 1) > 0.1   # rounded to nearest it would not have moved


# ---------------------------------------------------------------- lists, layouts, streams
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_of_several_kinds(bits):
    """More tensors than one launch takes, all types mixed: each as by itself."""
    g = torch.Generator().manual_seed(1)
    sizes = torch.randint(1, 700, (900,), generator=g).tolist()
    lists = [make(sizes[k::3], pt, bits=bits, master=master, seed=k)
             for k, (pt, master) in enumerate(((F32, False), (BF16, True), (F16, False)))]
    lists[2]["m"][:50], lists[2]["v"][:50] = zip(*[new_state(p)[:2] for p in lists[2]["p"][:50]])
    alone = copy.deepcopy(lists)
    every = {k: [x for tensors in zip(*(l[k] for l in lists)) for x in tensors] for k in lists[0]}
    call(every, count(7))
    for l, a in zip(lists, alone):
        for i in range(len(a["p"])):
            one = {k: [x[i]] for k, x in a.items()}
            call(one, count(7))
            for k in ("p", "m", "v", "master"):
                assert torch.equal(bits_of(l[k][i]), bits_of(one[k][0]))


def bits_of(t):
    return t.contiguous().reshape(-1).view(torch.uint8)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt", [F32, BF16])
def test_misaligned_and_strided(pt, bits):
    """Tensors that start anywhere, and gradients in another order."""
    base = make([3000], pt, bits=bits, master=True)
    want = copy.deepcopy(base)
    call(want, count())
    moved = {}
    for k, (x,) in base.items():
        n = x.numel()
        if k == "exponents" or n == 0:
            moved[k] = [x]
            continue
        room = torch.zeros(n + 5, dtype=x.dtype, device=dev)
        room[3:3 + n].copy_(x)
        moved[k] = [room[3:3 + n]]
    call(moved, count())
    for k in ("p", "m", "v"):
        assert torch.equal(bits_of(moved[k][0]), bits_of(want[k][0]))
    two = copy.deepcopy(base)
    for k in ("p", "g", "m", "v"):
        two[k] = [two[k][0].view(50, 60)]
    if two["master"][0].numel():
        two["master"] = [two["master"][0].view(50, 60)]
    two["g"] = [two["g"][0].t().contiguous().t()]
    call(two, count())
    assert torch.equal(bits_of(two["p"][0]), bits_of(want["p"][0]))


def test_neighbours_are_left_alone():
    """A view's surroundings keep their values, in every buffer."""
    for bits in (32, 8):
        room = {k: torch.full((1000,), 1, device=dev).to(t) for k, t in
                (("p", BF16), ("m", torch.float8_e4m3fn if bits == 8 else F32),
                 ("v", torch.float8_e4m3fn if bits == 8 else F32), ("master", F32))}
        e = torch.full((8, 2), 1, dtype=torch.uint8, device=dev)
        old = {k: x.clone() for k, x in room.items()}
        part = {k: [x[16:16 + 301]] for k, x in room.items()}
        part["g"] = [torch.ones(301, device=dev)]
        part["exponents"] = [e[2:4]] if bits == 8 else []
        call(part, count())
        for k, x in room.items():
            keep = torch.ones(1000, dtype=torch.bool, device=dev)
            keep[16:317] = False
            assert torch.equal(bits_of(x.float()[keep]), bits_of(old[k].float()[keep]))
        assert (e[:2] == 1).all() and (e[4:] == 1).all()


def test_empty_lists():
    step = count()
    assert adamw_step([], [], [], [], step, lr=1e-3) is None and step.item() == 1
    assert adamw_step([], [], [], [], step, lr=1e-3, max_norm=1.0).item() == 0 and step.item() == 2


def test_not_finite():
    """With a norm: nothing happens.  Without: as IEEE has it, and a group of 8-bit states reads back as NaN."""
    for bad in (float("nan"), float("inf")):
        for bits in (32, 8):
            l = make([600, 40], F32, bits=bits)
            l["g"][0][300] = bad
            old = copy.deepcopy(l)
            step = count(2)
            assert not torch.isfinite(call(l, step, max_norm=1.0))
            assert step.item() == 2
            assert all(torch.equal(bits_of(a), bits_of(b)) for k in l for a, b in zip(l[k], old[k]))
            call(l, step)
            assert step.item() == 3 and not torch.isfinite(l["p"][0][300]) and torch.isfinite(l["p"][1]).all()
            if bits == 8:
                m, v = dequantise(l["m"][0], l["v"][0], l["exponents"][0])
                assert torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
                assert torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all()
                call(l, step)
                assert torch.isnan(l["p"][0][256:512]).all() and torch.isfinite(l["p"][0][:256]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """A captured step, replayed, is the next step: count, learning rate and dither come from the device."""
    l = make([5000, 33], BF16, bits=bits, master=True)
    want = copy.deepcopy(l)
    step, lr = count(), torch.full((), 1e-2, device=dev)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        norm = call(l, step, lr=lr, max_norm=0.5)
    assert step.item() == 0
    eager = count()
    for t in range(4):
        rate = 1e-2 / (t + 1)
        lr.fill_(rate)
        for a, b in zip(l["g"], want["g"]):
            a.mul_(0.7), b.mul_(0.7)
        graph.replay()
        n2 = call(want, eager, lr=torch.full((), rate, device=dev), max_norm=0.5)
        assert torch.equal(norm, n2)
    assert step.item() == 4
    assert all(torch.equal(bits_of(a), bits_of(b)) for k in l for a, b in zip(l[k], want[k]))


def test_refusals():
    l = make([64, 32], BF16, master=True)
    ok = lambda: [l[k] for k in ("p", "g", "m", "v")]  # noqa: E731

    def refused(*lists, **kw):
        with pytest.raises((RuntimeError, ValueError)):
            adamw_step(*lists, kw.pop("step", count()), **{"lr": 1e-3, **kw})

    p, g, m, v = ok()
    before = [x.clone() for x in p]
    refused(p, g[:1], m, v)
    refused([p[0], p[0]], [g[0], g[0]], [m[0], m[0].clone()], [v[0], v[0].clone()])   # the same parameter twice
    refused([p[0][:40], p[0][30:62]], [g[0][:40], g[0][30:62]], [m[0][:40], m[0][30:62]], [v[0][:40], v[0][30:62]])
    refused(p, [x.half() for x in g], m, v)
    refused(p, [x[:5] for x in g], m, v)
    refused(p, g, [x.bfloat16() for x in m], v)
    refused(p, g, [x.to(torch.float8_e4m3fn) for x in m], [x.to(torch.float8_e4m3fn) for x in v])   # no exponents
    refused(p, g, m, v, masters=[x.float()[:3] for x in p])
    refused([x.float() for x in p], [x.float() for x in g], m, v, masters=[x.float() for x in p])
    refused(p, g, m, v, step=torch.zeros((), device=dev))
    refused(p, g, m, v, step=torch.zeros((), dtype=torch.int64))
    refused(p, g, m, v, betas=(1.0, 0.9))
    refused(p, g, m, v, max_norm=-1.0)
    refused(p, g, m, v, lr=torch.full((), 1e-3))
    refused([x.cpu() for x in p], g, m, v)
    refused([p[0].view(8, 8).t()], [g[0].view(8, 8)], [m[0].view(8, 8)], [v[0].view(8, 8)])
    assert all(torch.equal(a, b) for a, b in zip(p, before)) and _ext.device_status() == 0


def test_modes_and_subclasses_reach_the_operator():
    """Lists go past the dispatcher only where nothing there would see to them; either way the bits are the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.ops.append(func._opname)
            return func(*args, **(kwargs or {}))

    class Named(torch.Tensor):
        pass

    want, moded, named, tupled = (make([300, 20], BF16, master=True, bits=8) for _ in range(4))
    call(want, count())
    with Seen():
        call(moded, count())
    assert "adamw_step" in Seen.ops
    named["p"] = [x.as_subclass(Named) for x in named["p"]]
    call(named, count())
    call({k: tuple(v) for k, v in tupled.items()}, count())
    for l in (moded, named, tupled):
        assert all(torch.equal(bits_of(a), bits_of(b)) for k in want for a, b in zip(l[k], want[k]))
    compiled = make([300, 20], BF16, master=True, bits=8)
    torch.compile(lambda: call(compiled, count()))()
    assert all(torch.equal(bits_of(a), bits_of(b)) for k in want for a, b in zip(compiled[k], want[k]))


# ---------------------------------------------------------------- the optimizer
def small_model(dtype=F32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(70, 90), torch.nn.Tanh(), torch.nn.Linear(90, 3)).to(dev, dtype)


def train(model, opt, steps, start=0):
    for k in range(start, start + steps):
        x = torch.randn(16, 70, generator=torch.Generator().manual_seed(k)).to(dev, next(model.parameters()).dtype)
        opt.zero_grad(set_to_none=True)
        model(x).square().mean().backward()
        opt.step()
    return model


def test_optimizer_against_torch():
    """Ten fp32 steps beside torch.optim.AdamW with clipping: each step moves a parameter by at most about lr, with
    an error of 2^-20 of that, and the gradients that follow differ by as little; 10 lr 2^-16 bounds it."""
    ours, theirs = small_model(), small_model()
    a = AdamW(ours.parameters(), lr=1e-2, weight_decay=0.1, max_norm=0.05)
    b = torch.optim.AdamW(theirs.parameters(), lr=1e-2, weight_decay=0.1)
    for k in range(10):
        train(ours, a, 1, k)
        x = torch.randn(16, 70, generator=torch.Generator().manual_seed(k)).to(dev)
        b.zero_grad(set_to_none=True)
        theirs(x).square().mean().backward()
        norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), 0.05)
        assert abs(a.grad_norm[0] - norm) <= 1e-4 * norm
        b.step()
        # (where a gradient is as good as zero its sign decides the step: the moments' ratio is not continuous there)
    off = torch.cat([(x - y).abs().flatten() for x, y in zip(ours.parameters(), theirs.parameters())])
    assert (off <= 10 * 1e-2 * 2 ** -16).float().mean() > 0.999 and off.max() <= 2 * 10 * 1e-2


@pytest.mark.parametrize("bits,master", [(32, False), (8, True)])
def test_state_dict_goes_on_with_the_same_bits(bits, master):
    kw = dict(lr=1e-2, bits=bits, master=master, min_8bit_size=100)
    whole = small_model(BF16)
    train(whole, AdamW(whole.parameters(), **kw), 6)
    first = small_model(BF16)
    opt = AdamW(first.parameters(), **kw)
    train(first, opt, 3)
    saved = copy.deepcopy(opt.state_dict())
    second = small_model(BF16)
    second.load_state_dict(first.state_dict())
    opt2 = AdamW(second.parameters(), **kw)
    opt2.load_state_dict(saved)
    for p, q in zip(first.parameters(), second.parameters()):
        for key, value in opt.state[p].items():
            assert opt2.state[q][key].dtype == value.dtype and torch.equal(bits_of(opt2.state[q][key]), bits_of(value))
    train(second, opt2, 3, 3)
    assert all(torch.equal(a, b) for a, b in zip(whole.parameters(), second.parameters()))


def test_optimizer_groups_and_missing_gradients():
    model = small_model(BF16)
    ps = list(model.parameters())
    frozen = ps[1].detach().clone()
    opt = AdamW([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.5, "bits": 8}], lr=1e-3)
    ps[1].requires_grad_(False)
    version = ps[0]._version
    train(model, opt, 2)
    assert torch.equal(ps[1], frozen) and opt.grad_norm == [None, None] and ps[0]._version > version
    assert opt.state[ps[2]]["exp_avg"].dtype == torch.float32   # too small for 8 bits
    assert opt.param_groups[0]["step"].item() == 2
    with pytest.raises(ValueError):
        AdamW(ps, bits=16)
    with pytest.raises(ValueError):
        AdamW(ps, lr=-1.0)


def test_whole_training_step_in_a_graph():
    """Forward, backward and update captured together: replays train as eager steps do."""
    eager, graphed = small_model(), small_model()
    x = torch.randn(16, 70, device=dev)
    a = AdamW(eager.parameters(), lr=1e-2, max_norm=0.1)
    with pytest.raises(RuntimeError, match="init_states"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            for p in graphed.parameters():
                p.grad = torch.zeros_like(p)
            AdamW(graphed.parameters()).step()
    graphed = small_model()
    b = AdamW(graphed.parameters(), lr=1e-2, max_norm=0.1).init_states()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):   # (library handles are made outside the capture)
        graphed(x).square().mean().backward()
        for p in graphed.parameters():
            p.grad = None
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        graphed(x).square().mean().backward()
        b.step()
        for p in graphed.parameters():
            p.grad = None
    for _ in range(5):
        graph.replay()
        a.zero_grad(set_to_none=True)
        eager(x).square().mean().backward()
        a.step()
    assert b.param_groups[0]["step"].item() == 5
    assert all(torch.equal(p, q) for p, q in zip(eager.parameters(), graphed.parameters()))
