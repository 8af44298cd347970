"""Gradients of rmsnorm for rows of very large and very small magnitude, against the oracle in float64: the tolerances
are those of ordinary rows, and all rows of a case have the same magnitude."""
import pytest
import torch

from oracle import ops as O
from oracle.compare import norm_max_err

pytestmark = pytest.mark.gpu
dev = "cuda"


# a warp a row with the next one staged, a warp a row in fp32, a block a row, and rows of single values
@pytest.mark.parametrize("dt,d", [(torch.bfloat16, 1152), (torch.float32, 1152), (torch.bfloat16, 6000), (torch.float32, 77)])
@pytest.mark.parametrize("rms,eps", [(1e12, 1e-6), (1e15, 1e-6), (1e17, 1e-6), (1e-13, 1e-30)])
@pytest.mark.parametrize("added", [False, True])
def test_rows_of_any_magnitude(dt, d, rms, eps, added):
    import rmsnorm  # noqa: F401  (registers the operators)

    x, w, g = O.rmsnorm_inputs(37, d, torch.float32, seed=d)
    x, w, g, ga = (x * rms).to(dt), w.to(dt), g.to(dt), (O.gen((37, d), 3) / rms).to(dt)
    y, rstd = torch.ops.krsi.rmsnorm_fwd(x.to(dev), w.to(dev), eps)
    y_o, r_o = O.rmsnorm_fwd(x, w, eps)
    dx_o, dw_o = O.rmsnorm_bwd(g, x, w, r_o)
    if added:
        dx, dw = torch.ops.krsi.rmsnorm_bwd_add(g.to(dev), x.to(dev), w.to(dev), rstd, ga.to(dev))
        dx_o = dx_o.double() + ga.double()
    else:
        dx, dw = torch.ops.krsi.rmsnorm_bwd(g.to(dev), x.to(dev), w.to(dev), rstd)
    tol = 1e-5 if dt == torch.float32 else 1e-2
    assert norm_max_err(y.cpu(), y_o) <= tol
    assert norm_max_err(dx.cpu(), dx_o) <= tol
    assert norm_max_err(dw.cpu(), dw_o) <= tol
