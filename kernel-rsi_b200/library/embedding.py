"""The embedding lookup with scaling on B200 (hand-written sm_100a CUDA), and its gradient by sorted
tokens. Use embedding(tokens, table, scale, padding_idx).

embedding(tokens, table, scale=1.0, padding_idx=None) -> scale * table[tokens], [*tokens.shape, d]
  tokens: int32 or int64 of any shape; table: [V, d], fp32, bf16 or f16; the product is rounded once.
The backward returns the table's dense gradient: scale times the sum of the output's gradient rows of
each token, in fp32 in a fixed order over the positions sorted by token (no atomics: the same bits on
every run), rounded once.  padding_idx (negative counts from the end, as in torch) names a token whose
row gets no gradient; it is looked up like any other.

A token outside [0, V) cannot raise without a synchronisation: its row of the output is NaN and it adds
to no gradient.  The reference has no such op (its models use torch's embedding).
The autograd node is in csrc/torch_ext.cpp (krsi::embedding).
Kernels: kernel-rsi_b200/csrc/embedding.cu, token_rows.cu; C ABI: include/krsi_b200.h.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tools"))   # the skill's tools (selftest)
sys.path.insert(0, str(Path(__file__).resolve().parent))
from _compat import compiling  # noqa: E402
from _ext import ops  # noqa: E402


def embedding(tokens, table, scale=1.0, padding_idx=None):
    """scale * table[tokens] for integer tokens of any shape and a [V, d] table."""
    if padding_idx is None:
        pad = -1
    else:
        V = table.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} is outside a table of {V} rows")
        pad = padding_idx % V
    if compiling():
        return ops.embedding_fwd(tokens, table, scale, pad)
    return ops.embedding(tokens, table, scale, pad)


def reference(tokens, table, scale=1.0, padding_idx=None):
    """The torch expression this op reproduces."""
    return torch.nn.functional.embedding(tokens, table, padding_idx=padding_idx) * scale


def selftest():
    """The library's self-test contract (output and table gradient, eager and compiled) at 4096 tokens
    of a 32,768-row table."""
    from common import selftest_autograd  # noqa: PLC0415

    tokens = torch.randint(0, 32768, (4, 1024), device="cuda")
    table = torch.randn(32768, 768, device="cuda", dtype=torch.bfloat16)
    return selftest_autograd(lambda t: embedding(tokens, t, 0.5), lambda t: reference(tokens, t, 0.5), [table])


if __name__ == "__main__":
    print(selftest())
