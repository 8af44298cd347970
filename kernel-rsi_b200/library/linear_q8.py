"""A projection whose input and weight are in 8 bits, on B200 (a hand-written tcgen05 GEMM on the 8-bit tensor-core
rate). Use linear_q8(q, scale, wq, wscale, dtype) with quantise(w) and add_rmsnorm.add_rmsnorm_q8().

linear_q8(q, scale, wq, wscale, dtype)[i, j] = (sum over k of q[i, k] * wq[j, k]) * scale[i] * wscale[j] for
q [rows, K] and wq [M, K] in float8_e4m3fn and fp32 scales, one a row of each; summed in fp32, rounded once to
dtype (bf16, f16 or fp32).  Any K and M; rows that do not start on 16 bytes are copied first (quantise() and
add_rmsnorm_q8() pad theirs).

quantise(x2d) -> (q, scale): rows in 8 bits, the largest magnitude of each at 448: q = e4m3(x * (448 / m)),
scale = m / 448.  For weights, once: wq, wscale = quantise(linear.weight).

Against the same projection in bf16 the 8-bit operands cost 2^-4 of each value at most (3 bits of mantissa), about
2^-5.2 of the product's norm for normal operands.  Neither function has a gradient; both refuse to be called where
one could be asked for.
Kernels: kernel-rsi_b200/csrc/linear_q8.cu and csrc/add_rmsnorm.cu; C ABI: include/krsi_b200.h.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
from _ext import ops  # noqa: E402


def linear_q8(q, scale, wq, wscale, dtype=torch.bfloat16):
    """(q * scale[:, None]) @ (wq * wscale[:, None]).t() in dtype."""
    return ops.linear_q8(q, scale, wq, wscale, dtype)


def quantise(x2d):
    """(q, scale): the rows of x2d in 8 bits, x2d = q * scale[:, None] to within half a code."""
    return ops.quantise_rows(x2d)


def dequantise(q, scale):
    """The values that 8-bit rows stand for, in fp32 (torch ops)."""
    return q.float() * scale[:, None]


def reference(q, scale, wq, wscale, dtype=torch.bfloat16):
    """The torch expression linear_q8 replaces."""
    return ((q.float() @ wq.float().t()) * scale[:, None] * wscale).to(dtype)


def selftest():
    """linear_q8 against its torch expression at a gate|value projection's shape: the norm of the difference over the
    result's norm, which is the rounding to bf16 of either."""
    q, scale = quantise(torch.randn(2048, 768, device="cuda"))
    wq, wscale = quantise(torch.randn(4096, 768, device="cuda") * 768 ** -0.5)
    ref = reference(q, scale, wq, wscale, torch.float32)
    err = ((linear_q8(q, scale, wq, wscale).float() - ref).norm() / ref.norm()).item()
    return {"ok": err < 2 ** -8, "rel": err}


if __name__ == "__main__":
    print(selftest())
