"""add_rmsnorm and add_rmsnorm_q8 against their formulas in float64, and at the sizes, types and layouts where they
can go wrong.

Tolerances: u is half a step of a type relative to the value (torch.finfo(t).eps / 2).  z is exact (one rounding,
done alike).  y, dz and dw are rounded once; fp32 sums of k terms in chains of at most k / 32 + 32 are off by that many
2^-24 of the sum of magnitudes."""
import ctypes

import pytest
import torch

import _ext
from add_rmsnorm import add_rmsnorm, add_rmsnorm_q8
from gpu_util import DT, capi, ptr, stream
from linear_q8 import dequantise

pytestmark = pytest.mark.gpu
dev = "cuda"
EPS = 1e-6
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]
# rows of one packet, below and above a warp's and a block's plans, odd ones, and the widest of the scalar path
SHAPES = [(1, 1), (3, 7), (2, 8), (65, 250), (300, 1152), (33, 1149), (17, 2740), (5, 5000), (2, 9001), (3, 16384)]


def u(t):
    return torch.finfo(t).eps / 2


def inputs(n, d, dt, wt, seed=0, res=True):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, r, w = rand(n, d), rand(n, d) * torch.exp(rand(n, 1)), 1 + 0.1 * rand(d)
    gy, gz = rand(n, d), rand(n, d)
    return [t.to(dev, dt) for t in (x, r)] + [w.to(dev, wt)] + [t.to(dev, dt) for t in (gy, gz)]


def formula(z, w, gy, gz):
    """y, dz, dw in float64 for a rounded z, and the magnitudes that their errors are relative to."""
    z, w, gy = z.double(), w.double(), gy.double()
    r = 1 / torch.sqrt(z.square().mean(1, keepdim=True) + EPS)
    n = z * r
    gw = gy * w
    dz = r * gw - n * r * (gw * n).mean(1, keepdim=True)
    size = r * gw.abs() + n.abs() * r * (gw * n).abs().mean(1, keepdim=True)
    if gz is not None:
        dz, size = dz + gz.double(), size + 2 ** -24 * gz.double().abs()
    return n * w, dz, (gy * n).sum(0), size, (gy * n).abs().sum(0)


def check(z, w, gy, gz, y, dz, dw):
    y64, dz64, dw64, size, dw_size = formula(z, w, gy, gz)
    d32 = (z.shape[1] / 32 + 64) * 2 ** -24
    rows32 = (z.shape[0] + 64) * 2 ** -24
    ux, uw = u(z.dtype), u(w.dtype)
    low = torch.finfo(z.dtype).tiny * torch.finfo(z.dtype).eps
    assert ((y.double() - y64).abs() <= y64.abs() * (1.01 * ux + d32) + low).all()
    if dz is not None:
        assert ((dz.double() - dz64).abs() <= 1.01 * ux * dz64.abs() + 2 * d32 * size + low).all()
        assert ((dw.double() - dw64).abs() <= 1.01 * uw * dw64.abs() + (d32 + rows32) * dw_size + low).all()


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("n,d", SHAPES)
def test_step_against_float64(n, d, dt, wt):
    x, res, w, gy, gz = inputs(n, d, dt, wt)
    args = [t.clone().requires_grad_(True) for t in (x, res, w)]
    y, z = add_rmsnorm(*args, EPS)
    dx, dres, dw = torch.autograd.grad((y, z), args, (gy, gz))
    assert torch.equal(z, x + res) and y.dtype == dt
    check(z, w, gy, gz, y, dx, dw)
    assert torch.equal(dx, dres) and dw.dtype == wt
    with torch.no_grad():
        y2, z2 = add_rmsnorm(x, res, w, EPS)
    assert torch.equal(y, y2) and torch.equal(z, z2)


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("n,d", [(3, 7), (300, 1152), (17, 2740)])
def test_without_a_residual(n, d, dt, wt):
    """z is x; its gradient is added to the norm's."""
    x, _, w, gy, gz = inputs(n, d, dt, wt)
    args = [t.clone().requires_grad_(True) for t in (x, w)]
    y, z = add_rmsnorm(args[0], None, args[1], EPS)
    dx, dw = torch.autograd.grad((y, z), args, (gy, gz))
    assert torch.equal(z, x)
    check(x, w, gy, gz, y, dx, dw)


def test_either_gradient_alone():
    x, res, w, gy, gz = inputs(33, 72, BF16, BF16)
    args = [t.clone().requires_grad_(True) for t in (x, res, w)]
    y, z = add_rmsnorm(*args, EPS)
    dx, dres, first = torch.autograd.grad(y, args, gy, retain_graph=True)
    check(z, w, gy, None, y, dx, first)
    dx, dres, dw = torch.autograd.grad(z, args, gz, retain_graph=True, allow_unused=True)
    assert torch.equal(dx, gz) and torch.equal(dres, gz) and (dw is None or not dw.any())
    (dw1,) = torch.autograd.grad(y, args[2:], gy)   # the weight alone
    assert torch.equal(dw1, first)


def test_gradient_against_differences():
    """The kernel's gradient (fp32) in random directions against central differences of the formula in float64:
    their truncation is h^2 times a third derivative (about 1e-8 here), the kernel's error 1e-6 of the sizes."""
    x, res, w, gy, gz = inputs(5, 40, F32, F32)
    args = [t.clone().requires_grad_(True) for t in (x, res, w)]
    grads = torch.autograd.grad(add_rmsnorm(*args, EPS), args, (gy, gz))

    def loss(x, res, w):
        z = x + res
        y = z / torch.sqrt(z.square().mean(1, keepdim=True) + EPS) * w
        return (gy.double() * y + gz.double() * z).sum()

    base = [t.double() for t in (x, res, w)]
    for k in range(3):
        way = torch.randn_like(base[k])
        h = 1e-4
        up, down = ([t + s * h * way if i == k else t for i, t in enumerate(base)] for s in (1, -1))
        want = (loss(*up) - loss(*down)) / (2 * h)
        got = (grads[k].double() * way).sum()
        assert abs(got - want) <= 1e-5 * (grads[k].double() * way).abs().sum() + 1e-6


def test_layouts_and_streams():
    """Strided and misaligned operands and gradients, a stream of the caller's own, the same operand twice."""
    x, res, w, gy, gz = inputs(40, 264, BF16, BF16)
    with torch.no_grad():
        want = add_rmsnorm(x, res, w, EPS)
        wide = torch.zeros(40, 300, dtype=BF16, device=dev)
        for at in (0, 3):
            wide[:, at:at + 264] = x
            assert all(torch.equal(a, b) for a, b in zip(add_rmsnorm(wide[:, at:at + 264], res, w, EPS), want))
        flat = torch.zeros(40 * 264 + 3, dtype=BF16, device=dev)
        flat[3:] = res.reshape(-1)   # contiguous, off 16 bytes
        assert all(torch.equal(a, b) for a, b in zip(add_rmsnorm(x, flat[3:].view(40, 264), w, EPS), want))
        twice = add_rmsnorm(x, x, w, EPS)
        assert torch.equal(twice[1], x + x)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = add_rmsnorm(x, res, w, EPS)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    args = [t.clone().requires_grad_(True) for t in (x, res, w)]
    out = add_rmsnorm(*args, EPS)
    want = torch.autograd.grad(out, args, (gy, gz), retain_graph=True)
    odd = torch.zeros(40 * 264 + 1, dtype=BF16, device=dev)
    odd[1:] = gz.reshape(-1)
    gy_t = gy.t().contiguous().t()
    got = torch.autograd.grad(out, args, (gy_t, odd[1:].view(40, 264)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_same_operand_twice():
    """x as its own residual: both gradients reach it."""
    x, _, w, gy, gz = inputs(40, 264, BF16, BF16)
    leaf, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y, z = add_rmsnorm(leaf, leaf, lw, EPS)
    (dx,) = torch.autograd.grad((y, z), leaf, (gy, gz))
    _, dz, _, size, _ = formula(z, w, gy, gz)
    ux = u(BF16)   # dz is rounded once, twice it once more
    assert ((dx.double() - 2 * dz).abs() <= 2.1 * 2 * ux * dz.abs() + 4 * (264 / 32 + 64) * 2 ** -24 * size + 1e-30).all()


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("off", [4, 8])
def test_c_abi_at_addresses_off_16_bytes(dt, wt, off):
    """Every operand, the weight among them, `off` bytes past a 16-byte boundary; rows of whole 8 bytes, and odd ones."""
    lib = capi()
    for n, d in ((5, 260), (5, 264), (3, 77)):
        x, res, w, gy, gz = inputs(n, d, dt, wt)

        def shifted(t):
            k = off // t.element_size()
            room = torch.zeros(t.numel() + k, dtype=t.dtype, device=dev)
            room[k:] = t.reshape(-1)
            return room[k:].view(t.shape)

        a = [shifted(t) for t in (x, res, w, gy, gz)]
        y, z, dz, dw = (shifted(torch.zeros_like(t)) for t in (x, x, x, w))
        rstd, scale = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
        q = shifted(torch.zeros(n, d, dtype=torch.uint8, device=dev))
        ws = torch.zeros(n * d, device=dev)
        i64, kinds = ctypes.c_int64, (ctypes.c_int64(n), ctypes.c_int64(d))
        eps = ctypes.c_float(EPS)
        assert lib.krsi_add_rmsnorm_fwd(*map(ptr, (a[0], a[1], a[2], z, y, rstd)), *kinds, eps, DT[dt], DT[wt], stream()) == 0
        assert lib.krsi_add_rmsnorm_bwd(*map(ptr, (a[3], a[4], z, a[2], rstd, dz, dw, ws)), ctypes.c_size_t(n * d * 4),
                                        *kinds, DT[dt], DT[wt], stream()) == 0
        assert torch.equal(z, x + res)
        check(z, w, gy, gz, y, dz, dw)
        assert lib.krsi_add_rmsnorm_q8_fwd(*map(ptr, (a[0], a[1], a[2], z, q)), i64(d), ptr(scale), *kinds, eps, DT[dt],
                                           DT[wt], stream()) == 0
        assert torch.equal(q, codes(z, w)[0].view(torch.uint8))
    torch.cuda.synchronize()


def test_empty():
    w = torch.ones(16, device=dev, requires_grad=True)
    x = torch.empty(0, 16, device=dev, requires_grad=True)
    y, z = add_rmsnorm(x, x.detach(), w, EPS)
    dx, dw = torch.autograd.grad((y, z), (x, w), (y.detach(), z.detach()))
    assert y.shape == z.shape == dx.shape == (0, 16) and not dw.any()
    q, scale, z = add_rmsnorm_q8(x.detach(), None, w.detach(), EPS)
    assert q.shape == (0, 16) and scale.shape == (0,)


def codes(z, w):
    """add_rmsnorm_q8's rule in fp32: the codes, and the row's largest magnitude."""
    t = z.float() * w.float()
    top = t.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    return (t * (448.0 / top)).to(torch.float8_e4m3fn), top[:, 0]


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("add", [True, False])
def test_8_bits(n, d, dt, wt, add):
    """The codes bit for bit, the scale to fp32's last bits, y within half a code."""
    x, res, w, _, _ = inputs(n, d, dt, wt)
    q, scale, z = add_rmsnorm_q8(x, res if add else None, w, EPS)
    assert torch.equal(z, x + res if add else x)
    want, top = codes(z, w)
    assert torch.equal(q.view(torch.uint8), want.contiguous().view(torch.uint8))
    z64 = z.double()
    r = 1 / torch.sqrt(z64.square().mean(1) + EPS)
    d32 = (d / 32 + 64) * 2 ** -24
    s64 = top.double() * r / 448
    assert ((scale.double() - s64).abs() <= s64 * d32).all()
    y64 = z64 * r[:, None] * w.double()
    off = (dequantise(q, scale).double() - y64).abs()
    assert (off <= y64.abs() * (2 ** -4 + 2 * d32) + s64[:, None] * (2 ** -10 * (1 + d32))).all()


def test_8_bits_of_extreme_rows():
    """Zeros, tiny and huge rows, one value alone, and rows that are not finite (their scale is not either)."""
    x = torch.zeros(7, 96, device=dev)
    x[1] = 1e-30
    x[2] = 1e18
    x[3, 5] = 3.0
    x[4, 7] = float("nan")
    x[5, 9] = float("inf")
    x[6] = torch.linspace(-1, 1, 96, device=dev)
    w = torch.ones(96, device=dev)
    q, scale, _ = add_rmsnorm_q8(x, None, w, EPS)
    y = dequantise(q, scale)
    assert not y[0].any() and torch.isfinite(scale[[0, 1, 2, 3, 6]]).all()
    assert not torch.isfinite(scale[4]) and not torch.isfinite(scale[5])
    assert not torch.isfinite(y[4]).any() and not torch.isfinite(y[5, 9])
    assert abs(y[2, 0].item() - 1) < 2 ** -4 and abs(y[3, 5].item() - 96 ** 0.5) < 2 ** -4 * 10 and not y[3, 6:].any()


def test_captured_and_replayed():
    """A whole step in a CUDA graph, replayed on new values, gives the eager step's bits."""
    x, res, w, gy, gz = inputs(300, 1152, BF16, BF16)
    args = [t.clone().requires_grad_(True) for t in (x, res, w)]

    def step():
        y, z = add_rmsnorm(*args, EPS)
        return (y.detach(), z.detach(), *torch.autograd.grad((y, z), args, (gy, gz)),
                *add_rmsnorm_q8(args[0].detach(), args[1].detach(), args[2].detach(), EPS))

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    for seed in (1, 2):
        new = inputs(300, 1152, BF16, BF16, seed)
        with torch.no_grad():
            for a, b in zip(args, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out, want))


def test_compiled():
    x, res, w, gy, gz = inputs(64, 200, BF16, BF16)
    fn = torch.compile(lambda a, b, c: add_rmsnorm(a, b, c, EPS), fullgraph=True)
    alone = torch.compile(lambda a, c: add_rmsnorm(a, None, c, EPS), fullgraph=True)
    args = [t.clone().requires_grad_(True) for t in (x, res, w)]
    want = add_rmsnorm(*args, EPS)
    gw = torch.autograd.grad(want, args, (gy, gz))
    got = fn(*args)
    gg = torch.autograd.grad(got, args, (gy, gz))
    assert all(torch.equal(a, b) for a, b in zip((*got, *gg), (*want, *gw)))
    y, z = alone(args[0], args[2])
    y1, _ = add_rmsnorm(args[0], None, args[2], EPS)
    assert torch.equal(y, y1)
    got = torch.autograd.grad((y, z), (args[0], args[2]), (gy, gz))
    check(x, w, gy, gz, y1, *got)


def test_refusals():
    x, res, w, gy, gz = inputs(8, 32, BF16, BF16)
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: add_rmsnorm(x, res[:4], w, EPS), lambda: add_rmsnorm(x, res.float(), w, EPS),
                 lambda: add_rmsnorm(x, res, w[:8], EPS), lambda: add_rmsnorm(x[0], res[0], w, EPS),
                 lambda: add_rmsnorm(x, res, w.half(), EPS), lambda: add_rmsnorm(x, res.cpu(), w, EPS),
                 lambda: add_rmsnorm(x.double(), None, w.double(), EPS),
                 lambda: add_rmsnorm(torch.zeros(2, 40000, device=dev), None, torch.ones(40000, device=dev), EPS),
                 lambda: add_rmsnorm_q8(leaf, res, w, EPS), lambda: add_rmsnorm_q8(x, leaf, w, EPS)):
        with pytest.raises(RuntimeError):
            call()
    y, _ = add_rmsnorm(leaf, res, w, EPS)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(y, leaf, gy, create_graph=True)
    import torch.autograd.forward_ad as fwd_ad
    with fwd_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
        add_rmsnorm(fwd_ad.make_dual(x, gy), res, w, EPS)
    assert _ext.device_status() == 0
