"""The residual's addition and RMSNorm in one pass on B200 (hand-written sm_100a CUDA), its output in the
input's type or in 8 bits. Use add_rmsnorm(x2d, res, w, eps), or add_rmsnorm_q8(...) before a product in 8 bits.

add_rmsnorm(x2d, res, w, eps) -> (y, z): z = x2d + res rounded to their type, y = w * z / sqrt(mean(z^2) + eps) in
fp32, rounded once (rmsnorm() rounds the normalised row to w's type before the product, as the reference does,
rmsnorm.py:22-31); so are the gradients.  z is the residual of the next junction; its gradient is added inside the norm's backward, so
no pass over memory is left for either sum.  With res None, z is x2d: what remains is that addition.  fp32, bf16 and
f16, w in the same type or fp32; rows up to 16384 elements (32768 for 16-bit types with rows of whole 16 bytes).

add_rmsnorm_q8(x2d, res, w, eps) -> (q, scale, z): y in 8 bits, y = q * scale[:, None], q in float8_e4m3fn with the
row's largest magnitude at 448 and one fp32 scale a row (z as above).  y is not rounded on the way:
q = e4m3(z * w * (448 / m)), scale = m * rstd / 448 for the row's largest |z * w| m, so q does not depend on the
statistics.  q's rows are padded to whole 16 bytes in memory, as linear_q8() reads them without a copy.  It has no
gradient, and refuses to be called where one could be asked for.

A row with a value that is not finite has a norm, or a scale, that is not finite either.
add_rmsnorm's autograd node is in csrc/torch_ext.cpp (krsi::add_rmsnorm).
Kernels: kernel-rsi_b200/csrc/add_rmsnorm.cu; C ABI: include/krsi_b200.h.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tools"))   # the skill's tools (selftest)
sys.path.insert(0, str(Path(__file__).resolve().parent))
from _compat import compiling  # noqa: E402
from _ext import ops  # noqa: E402


class PassNorm(torch.autograd.Function):
    """(rmsnorm(x2d), x2d) whose backward adds both gradients, for compiled graphs (an operator may not return its
    input; eager has the same as a node in C++)."""

    @staticmethod
    def forward(ctx, x2d, w, eps):
        y, _, rstd = ops.add_rmsnorm_fwd(x2d, None, w, eps)
        ctx.save_for_backward(x2d, w, rstd)
        return y, x2d.view_as(x2d)

    @staticmethod
    def backward(ctx, gy, gz):
        dz, dw = ops.add_rmsnorm_bwd(gy, gz, *ctx.saved_tensors)
        return dz, dw, None


def add_rmsnorm(x2d, res, w, eps):
    """(y, z) with z = x2d + res (x2d where res is None) and y = w * z / sqrt(mean(z^2) + eps), over the rows of 2-D
    tensors."""
    if compiling():
        return PassNorm.apply(x2d, w, eps) if res is None else ops.add_rmsnorm_fwd(x2d, res, w, eps)[:2]
    return ops.add_rmsnorm(x2d, res, w, eps)


def add_rmsnorm_q8(x2d, res, w, eps):
    """(q, scale, z): add_rmsnorm's y in 8 bits, y = q * scale[:, None], and z."""
    q, scale, z = ops.add_rmsnorm_q8(x2d, res, w, eps)
    return q, scale, (x2d if res is None else z)


def reference(x2d, res, w, eps):
    """The torch expression add_rmsnorm reproduces."""
    z = x2d if res is None else x2d + res
    zf = z.float()
    inv = torch.rsqrt(zf.square().mean(dim=-1, keepdim=True) + eps)
    return (w * (zf * inv)).to(x2d.dtype), z


def selftest():
    """The library's self-test contract: output (y + z, so that both carry a gradient) and gradients."""
    from common import selftest_autograd  # noqa: PLC0415

    x, res = (torch.randn(4096, 1024, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w = (1 + 0.1 * torch.randn(1024, device="cuda")).to(torch.bfloat16)
    return selftest_autograd(lambda *a: sum(add_rmsnorm(*a, 1e-6)), lambda *a: sum(reference(*a, 1e-6)), [x, res, w])


if __name__ == "__main__":
    print(selftest())
