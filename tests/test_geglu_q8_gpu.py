"""GEGLU with the 8-bit checkpoint (B200) against the definition in float64: the output from u, the
checkpoint bit for bit, the gradient at the checkpoint's values, and the feed-forward built on it."""
import math

import pytest
import torch

import _ext
from geglu_q8 import dequantise, feed_forward_q8, geglu_q8, reference

pytestmark = pytest.mark.gpu
dev = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def checkpoint(u):
    """(q, exponents) of the definition, in float64."""
    rows, F = u.shape[0], u.shape[1] // 2
    G = (F + 31) // 32
    h = torch.nn.functional.pad(u.double().view(rows, 2, F), (0, 32 * G - F)).view(rows, 2, G, 32)
    bad = ~torch.isfinite(h).all(3)
    top = torch.where(torch.isfinite(h), h, 0.0).abs().amax(3)
    e = torch.frexp(top)[1] - 1                     # floor(log2(top))
    e = torch.where(top > 0, e, -200).clamp(min=-120) - 6
    q = torch.ldexp(h, -e[..., None].double()).round().clamp(-127, 127)
    q = q.view(rows, 2, 32 * G)[:, :, :F].reshape(rows, 2 * F)
    ex = torch.where(bad, 255, e + 127)
    return q, ex.transpose(1, 2), bad


def gelu64(a):
    z2 = 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
    s = torch.sigmoid(z2)
    return a * s, s + a * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a * a)


def inputs(rows, F, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(rows, 2 * F, generator=g) * torch.exp(torch.randn(1, 2 * F, generator=g))
    return u.to(dtype), torch.randn(rows, F, generator=g).to(dtype)


def close(got, want, mag, dtype):
    """One rounding of the type, and 32 fp32 roundings of the terms' magnitude (the products and sums of a
    formula of about a dozen steps, the approximate exponential and reciprocal at a few units each, the
    exponential's argument up to 20 carrying its own rounding)."""
    err = (got.cpu().double() - want).abs()
    bound = UNIT[dtype] * 1.01 * want.abs() + 32 * 2.0 ** -24 * mag + TINY[dtype]
    assert torch.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,F", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 4608), (257, 100), (64, 2740), (130, 96),
                                    (7, 1000), (3, 6), (2, 2049)])
def test_forward_checkpoint_and_gradient(rows, F, dtype):
    u, g = inputs(rows, F, dtype, rows + F)
    out, q, ex = torch.ops.krsi.geglu_q8_fwd(u.to(dev), True)
    a, b = u.double()[:, :F], u.double()[:, F:]
    gel, _ = gelu64(a)
    close(out, gel * b, (a * b).abs(), dtype)
    wq, wex, _ = checkpoint(u)
    assert torch.equal(q.cpu().double(), wq) and torch.equal(ex.cpu().long(), wex.long())
    k = dequantise(q, ex).cpu().double()
    assert torch.all((k - u.double()).abs() <= step_bound(wex, F, rows))
    du, again = torch.ops.krsi.geglu_q8_bwd(g.to(dev), q, ex, True)
    ka, kb, gd = k[:, :F], k[:, F:], g.double()
    gel, slope = gelu64(ka)
    # the slope's terms: s and a s (1 - s) 2 dz/da, each of the order of 1
    close(du, torch.cat([gd * kb * slope, gd * gel], 1), torch.cat([2 * (gd * kb).abs(), (gd * ka).abs()], 1), dtype)
    close(again, gel * kb, (ka * kb).abs(), dtype)
    du2, none = torch.ops.krsi.geglu_q8_bwd(g.to(dev), q, ex, False)
    assert torch.equal(du, du2) and none.numel() == 0
    only, q0, ex0 = torch.ops.krsi.geglu_q8_fwd(u.to(dev), False)
    assert torch.equal(only, out) and q0.numel() == 0 and ex0.numel() == 0
    assert _ext.device_status() == 0


def step_bound(ex, F, rows):
    """One step (half a step, or up to one where the largest values round down to 127)."""
    step = torch.exp2(ex.double() - 127).transpose(1, 2).repeat_interleave(32, 2)[:, :, :F]
    return step.reshape(rows, 2 * F)


def test_ties_zeros_and_extremes():
    F = 32
    u = torch.zeros(6, 2 * F)
    u[1, :8] = torch.tensor([64.0, 0.5, 1.5, 2.5, -0.5, -1.5, 127.0, -127.0])      # ties to even, step 1
    u[2, :3] = torch.tensor([127.5, -127.75, 126.5])                                # past 127: held at 127
    u[3, :2] = torch.tensor([2.0 ** -140, -2.0 ** -126])                            # below the smallest step
    u[4, :2] = torch.tensor([3.0e38, -1.0])
    u[5, F:F + 2] = torch.tensor([2.0 ** -120, 2.0 ** -126])
    q, ex = torch.ops.krsi.geglu_q8_fwd(u.to(dev), True)[1:]
    wq, wex, _ = checkpoint(u)
    assert torch.equal(q.cpu().double(), wq) and torch.equal(ex.cpu().long(), wex.long())
    assert q[1, :8].tolist() == [64, 0, 2, 2, 0, -2, 127, -127] and q[2, :3].tolist() == [127, -127, 126]
    assert not q[0].any()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite_read_back_as_nan(bad):
    F = 64
    u, g = inputs(3, F, torch.float32, 1)
    u[1, 5] = bad                     # gate, group 0
    u[2, F + 40] = bad                # value, group 1
    q, ex = torch.ops.krsi.geglu_q8_fwd(u.to(dev), True)[1:]
    flagged = (ex == 255).cpu()
    assert flagged.sum() == 2 and flagged[1, 0, 0] and flagged[2, 1, 1]
    du = torch.ops.krsi.geglu_q8_bwd(g.to(dev), q, ex, False)[0].cpu()
    nan = torch.zeros(3, 2 * F, dtype=torch.bool)
    nan[1, :32] = nan[1, F:F + 32] = True            # both gradients of the gate's group
    nan[2, 32:64] = True                              # the gate's gradient takes the value
    assert torch.equal(du.isnan(), nan)


def test_large_gates_saturate():
    u = torch.tensor([[40.0, -40.0, 1e4, -1e4, 0.0, 1e30, -1e30, 3.0] * 4 + [1.0] * 32], device=dev)
    out = geglu_q8(u).cpu()[0]
    assert out[:3].tolist() == [40.0, 0.0, 1e4] and out[4] == 0 and out[3] == 0
    assert out[5] == u[0, 5].cpu() and out[6] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_huge_gates(dtype):
    """Gates whose square overflows fp32: the slope is 1 or 0 there, not 0 times infinity."""
    F = 32
    u = torch.ones(4, 2 * F)
    for r, big in enumerate((3e19, -3e19, 3e38, -3e38)):
        u[r, :F] = big
    x = u.to(dev, dtype).requires_grad_(True)
    (du,) = torch.autograd.grad(geglu_q8(x), x, torch.ones(4, F, device=dev, dtype=dtype))
    assert torch.equal(du[:, :F].cpu(), torch.tensor([1.0, 0, 1, 0], dtype=dtype)[:, None].expand(4, F))


def test_autograd_and_compile():
    u, g = inputs(40, 96, torch.bfloat16, 3)
    x = u.to(dev).requires_grad_(True)
    y = geglu_q8(x)
    (du,) = torch.autograd.grad(y, x, g.to(dev))
    out, q, ex = torch.ops.krsi.geglu_q8_fwd(u.to(dev), True)
    assert torch.equal(y.detach(), out) and torch.equal(du, torch.ops.krsi.geglu_q8_bwd(g.to(dev), q, ex, False)[0])
    z = torch.compile(geglu_q8, fullgraph=True)(x)
    assert torch.equal(z, y) and torch.equal(torch.autograd.grad(z, x, g.to(dev))[0], du)
    with torch.no_grad():
        assert torch.equal(geglu_q8(x), out)


def test_gradient_against_differences():
    """At values that the checkpoint holds exactly (integers up to 64 in a group led by 64) the gradient is
    GEGLU's own: central differences of the fp32 output with a step of 2^-6 have an error of order
    step^2 |f'''| / 6 (< 1e-4 here) and a rounding of 2^-24 |f| / step (< 4e-4 for |f| < 64)."""
    F = 32
    u = torch.randint(-3, 4, (4, 2 * F), generator=torch.Generator().manual_seed(0)).float()
    u[:, 31] = 64
    u[:, F + 31] = 64
    x = u.to(dev).requires_grad_(True)
    (du,) = torch.autograd.grad(geglu_q8(x), x, torch.ones(4, F, device=dev))
    h = 2.0 ** -6
    for col in (0, 7, F + 3, F + 30):
        step = torch.zeros_like(u)
        step[:, col] = h
        quot = (geglu_q8((u + step).to(dev)) - geglu_q8((u - step).to(dev))).sum(1) / (2 * h)
        assert (quot - du[:, col]).abs().max().item() < 1e-3


def test_feed_forward():
    """feed_forward_q8 against the same steps in float64 from the kernel's own checkpoint."""
    rows, d, F = 200, 128, 320
    gen = torch.Generator().manual_seed(5)
    x, wi, wo, res, gy = (torch.randn(*s, generator=gen) * k for s, k in
                          (((rows, d), 1.0), ((2 * F, d), d ** -0.5), ((d, F), F ** -0.5), ((rows, d), 1.0),
                           ((rows, d), 1.0)))
    args = [t.to(dev, torch.bfloat16).requires_grad_(True) for t in (x, wi, wo, res)]
    y = feed_forward_q8(*args)
    grads = torch.autograd.grad(y, args, gy.to(dev, torch.bfloat16))
    X, WI, WO, RES = (a.detach().cpu().double() for a in args)
    GY = gy.bfloat16().double()
    u = (args[0].detach() @ args[1].detach().t())
    out, q, ex = torch.ops.krsi.geglu_q8_fwd(u, True)
    k = dequantise(q, ex).cpu().double()
    gel, slope = gelu64(k[:, :F])
    dg = (GY @ WO).bfloat16().double()
    du = torch.cat([dg * k[:, F:] * slope, dg * gel], 1)
    want = [RES + out.cpu().double() @ WO.t(), du @ WI, du.t() @ X, GY.t() @ (gel * k[:, F:]), GY]
    for got, ref in zip([y.detach(), *grads], want):
        # bf16 operands (du, dg rounded once more than here) and one rounding of the result: 4 units of 2^-9
        # of the norm
        assert (got.cpu().double() - ref).norm() <= 4 * 2.0 ** -9 * ref.norm()
    y2 = feed_forward_q8(*args[:3])
    assert torch.allclose(y2.float(), (y - args[3]).float(), atol=0.1)


def test_checkpoint_keeps_training_close():
    """The gradient at the 8-bit values against the gradient at u itself: the checkpoint moves each value by
    at most 1/128 of its group's largest magnitude; over Gaussian groups of 32 (largest about 2.1 sigma)
    that is an rms of 2.1 / 64 / sqrt(12) = 0.9% of sigma, and GEGLU's gradient moves by the same order."""
    u, g = inputs(512, 512, torch.float32, 7)
    u = torch.randn(512, 1024, generator=torch.Generator().manual_seed(8))
    x = u.to(dev).requires_grad_(True)
    (du,) = torch.autograd.grad(geglu_q8(x), x, g.to(dev))
    (ref,) = torch.autograd.grad(reference(x), x, g.to(dev))
    assert ((du - ref).norm() / ref.norm()).item() < 0.03


def test_empty_and_refusals():
    for shape in ((0, 64), (4, 0)):
        x = torch.empty(shape, device=dev, requires_grad=True)
        y = geglu_q8(x)
        assert y.shape == (shape[0], shape[1] // 2)
        assert torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == shape
    with pytest.raises(RuntimeError, match="2F"):
        geglu_q8(torch.zeros(4, 7, device=dev))
    with pytest.raises(RuntimeError, match="dtype"):
        geglu_q8(torch.zeros(4, 8, device=dev, dtype=torch.float64))
    with pytest.raises((RuntimeError, NotImplementedError)):
        geglu_q8(torch.zeros(4, 8))
    q, ex = torch.ops.krsi.geglu_q8_fwd(torch.zeros(4, 64, device=dev), True)[1:]
    with pytest.raises(RuntimeError, match="g must be"):
        torch.ops.krsi.geglu_q8_bwd(torch.zeros(4, 31, device=dev), q, ex, False)
    with pytest.raises(RuntimeError, match="exponents"):
        torch.ops.krsi.geglu_q8_bwd(torch.zeros(4, 32, device=dev), q, ex[:3], False)
