"""Gradients of add_rmsnorm for rows of very large and very small magnitude, where powers of the row's 1 / rms leave
fp32's range although the gradients themselves do not.

Tolerances: dz and dw are rounded once (u: half a step of the type); fp32 sums of k terms in chains of at most
k / 32 + 32 are off by that many 2^-24 of the sum of magnitudes.  They hold at any scale: the formula's parts
z * r, mean(gy * w * z * r) and r * gy * w are all far from the ends of fp32's range here."""
import pytest
import torch

import _ext
from add_rmsnorm import add_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


# 16-bit rows of whole 16 bytes up to 1280 values have a kernel of their own; 2048, 1149 and fp32 take the other
@pytest.mark.parametrize("dt,d", [(BF16, 1152), (BF16, 40), (BF16, 2048), (BF16, 1149), (F32, 1152), (F32, 77)])
@pytest.mark.parametrize("rms,eps", [(1.0, 1e-6), (1e12, 1e-6), (1e15, 1e-6), (1e17, 1e-6), (1e-6, 1e-14), (1e-13, 1e-30)])
@pytest.mark.parametrize("g", [1.0, 1e-6])
@pytest.mark.parametrize("both", [True, False])
def test_rows_of_any_magnitude(dt, d, rms, eps, g, both):
    gen = torch.Generator().manual_seed(d)
    rand = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    x, res = (rand(29, d) * rms).to(dt), (rand(29, d) * rms).to(dt)
    w, gy, gz = (1 + 0.1 * rand(d)).to(dt), (rand(29, d) * g).to(dt), (rand(29, d) * (g / rms)).to(dt)
    args = [t.requires_grad_(True) for t in (x, res, w)]
    y, z = add_rmsnorm(*args, eps)
    dx, dres, dw = torch.autograd.grad((y, z) if both else y, args, (gy, gz) if both else gy)
    z64, w64, g64 = z.detach().double(), w.detach().double(), gy.double()
    r = 1 / torch.sqrt(z64.square().mean(1, keepdim=True) + eps)
    n, gw = z64 * r, g64 * w64
    want = r * (gw - n * (gw * n).mean(1, keepdim=True))
    size = r * (gw.abs() + n.abs() * (gw * n).abs().mean(1, keepdim=True))
    if both:
        want, size = want + gz.double(), size + 2 ** -24 * gz.double().abs()
    u, fi = torch.finfo(dt).eps / 2, torch.finfo(dt)
    d32, rows32, low = (d / 32 + 64) * 2 ** -24, (29 + 64) * 2 ** -24, fi.tiny * fi.eps
    assert ((dx.double() - want).abs() <= 1.01 * u * want.abs() + 2 * d32 * size + low).all()
    assert torch.equal(dx, dres)
    dw64, dw_size = (g64 * n).sum(0), (g64 * n).abs().sum(0)
    assert ((dw.double() - dw64).abs() <= 1.01 * u * dw64.abs() + (d32 + rows32) * dw_size + low).all()
    assert _ext.device_status() == 0
