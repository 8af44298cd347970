"""Softmax cross entropy of a projection onto the vocabulary on B200 (hand-written tcgen05 GEMMs), with
both gradients and without the [N, V] logits. Use linear_cross_entropy(x2d, w, targets, ...).

linear_cross_entropy(x2d, w, targets, scale=1.0, ignore_index=-100, z_loss=0.0, reduction="mean")
  x2d: [N, K]; w: [V, K] (the projection, or the tied embedding table); bf16 or f16, K a multiple of 8
  targets: [N] int32 or int64
  logits = scale * x2d @ w.t();  loss_i = logsumexp(logits_i) - logits_i[targets_i]
                                          + z_loss * logsumexp(logits_i)^2
  reduction: "mean" over the rows that are not ignored, "sum", or "none" ([N]); the result is fp32.
A row whose target is ignore_index has a loss and gradients of zero, whatever its x2d holds.  With
"mean" and no row left the loss is 0 and so are the gradients (torch's cross_entropy gives NaN there).
A target outside the vocabulary cannot raise without a synchronisation: it makes the loss and the
gradients NaN.

The logits exist one tile at a time, in the GEMM's epilogue.  With "mean" or "sum" and KEEP_ROWS rows
or more, the forward also forms both gradients (of the sum of the losses, in fp32) while the
exponentials are at hand, and the backward only scales and rounds them: one pass over the logits in all,
for the memory of two fp32 gradients.  Otherwise the backward computes the logits again.
Sums, statistics and the targets' own terms are fp32; the exponentials and the scaled rows of x that the
gradient products multiply are in the operands' 16 bits, so a row of dw whose token is no row's target
carries up to two roundings more than its result's own.
The reference has no loss op.  The autograd node is in csrc/torch_ext.cpp (krsi::linear_ce).
Kernels: kernel-rsi_b200/csrc/linear_ce.cu; C ABI: include/krsi_b200.h.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tools"))   # the skill's tools (selftest)
sys.path.insert(0, str(Path(__file__).resolve().parent))
from _compat import compiling  # noqa: E402
from _ext import ops  # noqa: E402

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
KEEP_ROWS = 1024


def linear_cross_entropy(x2d, w, targets, scale=1.0, ignore_index=-100, z_loss=0.0, reduction="mean"):
    """The cross entropy of softmax(scale * x2d @ w.t()) against targets, for x2d [N, K] and w [V, K]."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    kind = REDUCTIONS[reduction]
    keep = kind != 0 and x2d.shape[0] >= KEEP_ROWS
    if compiling():
        keep = keep and torch.is_grad_enabled()
        loss, total, *_ = ops.linear_ce_fwd(x2d, w, targets, scale, ignore_index, z_loss, kind,
                                                keep and x2d.requires_grad, keep and w.requires_grad)
        return total if kind else loss
    return ops.linear_ce(x2d, w, targets, scale, ignore_index, z_loss, kind, keep)


def reference(x2d, w, targets, scale=1.0, ignore_index=-100, z_loss=0.0, reduction="mean"):
    """The torch expression this op reproduces (it keeps the [N, V] logits)."""
    logits = (x2d.float() @ w.float().t()) * scale
    loss = torch.nn.functional.cross_entropy(logits, targets.long(), ignore_index=ignore_index, reduction="none")
    if z_loss:
        loss = loss + z_loss * torch.logsumexp(logits, 1).square() * (targets != ignore_index)
    if reduction == "none":
        return loss
    return loss.sum() / ((targets != ignore_index).sum().clamp(min=1) if reduction == "mean" else 1)


def selftest():
    """The library's self-test contract (loss and both gradients, eager and compiled) at 2048 rows of a
    base-size model's width over 32,768 entries."""
    from common import selftest_autograd  # noqa: PLC0415

    x = torch.randn(2048, 768, device="cuda", dtype=torch.bfloat16)
    w = (torch.randn(32768, 768, device="cuda") * 768 ** -0.5).to(torch.bfloat16)
    t = torch.randint(0, 32768, (2048,), device="cuda")
    return selftest_autograd(lambda x, w: linear_cross_entropy(x, w, t), lambda x, w: reference(x, w, t), [x, w])


if __name__ == "__main__":
    print(selftest())
