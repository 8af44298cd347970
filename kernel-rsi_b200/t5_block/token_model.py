"""A T5 encoder stack as a token model, on the library ops end to end: the masked positions of a token
sequence are predicted from the others, with one table for the way in and the way out.

  tokens    embedding(): the table's rows (entries of the order of d^-0.5), sqrt(d) times
  blocks    T5Block (model_entry.py) as in impl.py, its feed-forward on feed_forward_q8() (the
            projection kept in 8 bits for the backward) or feed_forward()
  final     rmsnorm()
  loss      linear_cross_entropy() of the rows on the same table, with z-loss; positions that are not
            predicted are ignored

  python kernel-rsi_b200/t5_block/token_model.py [--steps 40] [--layers 2] [--vocab 8192] [--batch 8]

trains it on synthetic sequences (each token follows from the one before) and prints the loss, the
tokens per second and the memory at its largest.
"""
import argparse
import math
import sys
import time
from pathlib import Path

import torch
from torch import nn

_HERE = Path(__file__).resolve().parent
for _p in (str(_HERE), str(_HERE.parent / "library")):
    if _p not in sys.path:
        sys.path.insert(0, _p)
import embedding  # noqa: E402
import geglu_q8  # noqa: E402
import linear_cross_entropy  # noqa: E402
import linear_geglu  # noqa: E402
import model_entry  # noqa: E402
import relpos_attention  # noqa: E402
import rmsnorm  # noqa: E402
import t5_bias  # noqa: E402

IGNORE = -100


def block(mod, x2, B, S, checkpoint8):
    """One T5Block on [B*S, d] rows."""
    H = mod.relative_attention_bias.weight.shape[1]
    D = mod.q.weight.shape[0] // H
    h = rmsnorm.rmsnorm(x2, mod.ln1.weight, mod.ln1.eps)
    qkv = h @ torch.cat([mod.q.weight, mod.k.weight, mod.v.weight]).t()
    pd = t5_bias.t5_relpos_bias(mod.relative_attention_bias.weight, S, True,
                                mod.relative_attention_bias.num_embeddings, 128)
    a = relpos_attention.relpos_attention(qkv, pd, B, S, H, D, 1.0)
    x2 = torch.addmm(x2, a, mod.o.weight.t())
    h = rmsnorm.rmsnorm(x2, mod.ln2.weight, mod.ln2.eps)
    ff = geglu_q8.feed_forward_q8 if checkpoint8 else linear_geglu.feed_forward
    return ff(h, torch.cat([mod.wi_0.weight, mod.wi_1.weight]), mod.wo.weight, x2)


class TokenModel(nn.Module):
    def __init__(self, vocab, layers=2, checkpoint8=True, z_loss=1e-4):
        super().__init__()
        self.table = nn.Parameter(torch.empty(vocab, model_entry.D_MODEL))
        self.layers = nn.ModuleList(model_entry.T5Block() for _ in range(layers))
        self.ln = model_entry.T5LayerNorm(model_entry.D_MODEL)
        self.checkpoint8, self.z_loss = checkpoint8, z_loss

    def forward(self, tokens, targets):
        """The mean loss over the positions whose target is not IGNORE; tokens, targets: [B, S]."""
        B, S = tokens.shape
        d = self.table.shape[1]
        x2 = embedding.embedding(tokens, self.table, scale=math.sqrt(d)).view(B * S, d)
        for layer in self.layers:
            x2 = block(layer, x2, B, S, self.checkpoint8)
        h = rmsnorm.rmsnorm(x2, self.ln.weight, self.ln.eps)
        return linear_cross_entropy.linear_cross_entropy(h, self.table, targets.reshape(-1),
                                                         ignore_index=IGNORE, z_loss=self.z_loss)

    def reference(self, tokens, targets):
        """The same model in torch (T5Block's own forward, torch's lookup, logits and cross entropy)."""
        d = self.table.shape[1]
        x = nn.functional.embedding(tokens, self.table) * math.sqrt(d)
        for layer in self.layers:
            x = layer(x)
        h = self.ln(x).reshape(-1, d)
        return linear_cross_entropy.reference(h, self.table, targets.reshape(-1), ignore_index=IGNORE,
                                              z_loss=self.z_loss)


def build(vocab, layers=2, checkpoint8=True, seed=0):
    model = TokenModel(vocab, layers, checkpoint8)
    model_entry.init_(model, seed)
    with torch.no_grad():
        g = torch.Generator().manual_seed(seed + 1)
        model.table.copy_(torch.randn(model.table.shape, generator=g) * model.table.shape[1] ** -0.5)
    return model.cuda().to(torch.bfloat16)


def batch(vocab, B, S, seed, device="cuda"):
    """Sequences in which each token follows from the one before (t -> 5 t + 3 mod 64, or mod the vocabulary
    less its mask token where that is smaller), 15% of them masked; the masked ones are the targets."""
    if vocab < 2:
        raise ValueError(f"a vocabulary of {vocab} has no token beside the mask token")
    used = min(64, vocab - 1)
    g = torch.Generator().manual_seed(seed)
    t = [torch.randint(0, used, (B,), generator=g)]
    for _ in range(S - 1):
        t.append((5 * t[-1] + 3) % used)
    tokens = torch.stack(t, 1)
    masked = torch.rand(B, S, generator=g) < 0.15
    targets = torch.where(masked, tokens, IGNORE)
    return torch.where(masked, vocab - 1, tokens).to(device), targets.to(device)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=8192)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--seq", type=int, default=512)
    ap.add_argument("--lr", type=float, default=1e-3)
    ap.add_argument("--no-checkpoint8", action="store_true", help="keep the feed-forward's activations in 16 bits")
    a = ap.parse_args(argv)
    model = build(a.vocab, a.layers, not a.no_checkpoint8)
    opt = torch.optim.AdamW(model.parameters(), lr=a.lr, weight_decay=0.0)
    losses = []
    torch.cuda.reset_peak_memory_stats()
    for step in range(a.steps):
        tokens, targets = batch(a.vocab, a.batch, a.seq, step)
        if step == min(3, a.steps - 1):
            torch.cuda.synchronize()
            began = time.perf_counter()
        loss = model(tokens, targets)
        loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(loss.detach())
    torch.cuda.synchronize()
    timed = a.steps - min(3, a.steps - 1)
    rate = timed * a.batch * a.seq / (time.perf_counter() - began)
    losses = torch.stack(losses).tolist()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps, {rate:,.0f} tokens/s, "
          f"{torch.cuda.max_memory_allocated() / 2 ** 20:,.0f} MiB")
    return losses


if __name__ == "__main__":
    main()
