"""GEGLU with an 8-bit checkpoint of its input on B200 (hand-written sm_100a CUDA): half the memory of
GEGLU's saved activation. Use geglu_q8(u), or feed_forward_q8(x2d, wi, wo, res).

geglu_q8(u) == gelu_tanh(u[:, :F]) * u[:, F:] for u [rows, 2F] (fp32, bf16 or f16), computed in fp32 and
rounded once (geglu() rounds gelu_tanh to the dtype before the product, as the reference does,
geglu.py:27-35).  Its backward does not keep u: the forward writes u in 8 bits, a signed byte per value
and, per group of 32 columns of a half-row, one byte of exponent (a step 2^-6 of the power of two at or
below the group's largest magnitude, values rounded to nearest even: at most 1/128 of that magnitude
off), and the backward is GEGLU's gradient at those values.  u itself is free once the forward has run:
8.25 bits a value are kept in place of 16 or 32.  A group with a value that is not finite reads back as
NaN.

feed_forward_q8(x2d, wi, wo, res) is res + geglu(x2d @ wi.t()) @ wo.t() that keeps x2d, the weights and
the checkpoint only: the GEGLU output, which the down projection's weight gradient needs, is computed
again from the checkpoint in the same pass as u's gradient.  Per row 2.06 F bytes stay for the backward
where feed_forward() keeps 6F (u and the GEGLU output in 16 bits), compiled or not.  The products are cuBLAS,
so that memory costs the fused GEMMs: a step of 32,768 x 1,152 x 4,608 takes 2.87 to 2.99 ms against 2.49 to
2.75, its forward alone 1.10 to 1.13 against 0.88 to 0.91 (B200, bf16).  Without a gradient to come neither
function writes a checkpoint.
geglu_q8's autograd node is in csrc/torch_ext.cpp (krsi::geglu_q8).
Kernels: kernel-rsi_b200/csrc/geglu_q8.cu; C ABI: include/krsi_b200.h.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tools"))   # the skill's tools (selftest)
sys.path.insert(0, str(Path(__file__).resolve().parent))
from _compat import compiling  # noqa: E402
from _ext import ops  # noqa: E402

GROUP = 32


def geglu_q8(u):
    """gelu_tanh(u[:, :F]) * u[:, F:] for u [rows, 2F], its backward from an 8-bit copy of u."""
    if compiling():
        return ops.geglu_q8_fwd(u, torch.is_grad_enabled() and u.requires_grad)[0]
    return ops.geglu_q8(u)


class FeedForwardQ8(torch.autograd.Function):
    """res + geglu(x2d @ wi^T) @ wo^T; saves (x2d, wi, wo, q, exponents); returns (dx, dwi, dwo, dres).
    keep: whether a gradient but res's can be asked for; else there is no checkpoint."""

    @staticmethod
    def forward(ctx, x2d, wi, wo, res, keep):
        g, q, ex = ops.geglu_q8_fwd(x2d @ wi.t(), keep)
        if keep:
            ctx.save_for_backward(x2d, wi, wo, q, ex)
        ctx.has_res = res is not None
        return torch.addmm(res, g, wo.t()) if res is not None else g @ wo.t()

    @staticmethod
    def backward(ctx, gy):
        if torch.is_grad_enabled():   # it would miss what du owes to gy and the operands
            raise RuntimeError("feed_forward_q8: the backward has no gradient of its own (create_graph)")
        if not any(ctx.needs_input_grad[:3]):
            return None, None, None, gy, None
        x2d, wi, wo, q, ex = ctx.saved_tensors
        gy = gy.contiguous()
        du, g = ops.geglu_q8_bwd(gy @ wo, q, ex, ctx.needs_input_grad[2])
        dx = du @ wi if ctx.needs_input_grad[0] else None
        dwi = du.t() @ x2d if ctx.needs_input_grad[1] else None
        dwo = gy.t() @ g if ctx.needs_input_grad[2] else None
        return dx, dwi, dwo, (gy if ctx.has_res else None), None


def feed_forward_q8(x2d, wi, wo, res=None):
    """res + geglu(x2d @ wi.t()) @ wo.t() for x2d [rows, d], wi [2F, d], wo [d, F] (and res [rows, d]),
    keeping the projection in 8 bits for the backward."""
    keep = torch.is_grad_enabled() and (x2d.requires_grad or wi.requires_grad or wo.requires_grad)
    return FeedForwardQ8.apply(x2d, wi, wo, res, keep)


def dequantise(q, exponents):
    """The values a checkpoint stands for, [rows, 2F] fp32 (torch ops; what the backward reads)."""
    rows, F = q.shape[0], q.shape[1] // 2
    step = torch.where(exponents == 255, float("nan"), torch.exp2(exponents.double() - 127))   # [rows, G, 2]
    step = step.transpose(1, 2).repeat_interleave(GROUP, dim=2)[:, :, :F]
    return (q.view(rows, 2, F).double() * step).view(rows, 2 * F).float()


def reference(u):
    """The torch expression this op reproduces (its gradient is at u, not at the 8-bit copy)."""
    gate, value = u.float().chunk(2, dim=-1)
    return (torch.nn.functional.gelu(gate, approximate="tanh") * value).to(u.dtype)


def selftest():
    """The library's self-test contract on u's that the checkpoint holds exactly (multiples of 1/16 with
    every group's largest magnitude between 4 and 8: within 127 steps), so output and gradient are those
    of the torch expression."""
    from common import selftest_autograd  # noqa: PLC0415

    u = (torch.randn(2048, 2 * 2048, device="cuda").clamp(-4, 4) * 16).round() / 16
    u[:, ::GROUP] = 4.0
    return selftest_autograd(geglu_q8, reference, [u.to(torch.bfloat16)])


if __name__ == "__main__":
    print(selftest())
