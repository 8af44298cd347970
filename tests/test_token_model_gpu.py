"""The token model (kernel-rsi_b200/t5_block/token_model.py): embedding, blocks, 8-bit feed-forward
checkpoint and vocabulary cross entropy together, against the same model in torch in fp32."""
import copy
import importlib.util

import pytest
import torch

import _ext
from conftest import PKG

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tm():
    spec = importlib.util.spec_from_file_location("krsi_token_model", PKG / "t5_block" / "token_model.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def step(model, fn, tokens, targets):
    ps = list(model.parameters())
    loss = fn(tokens, targets)
    return loss.detach(), [p.float() for p in torch.autograd.grad(loss, ps)]


@pytest.mark.parametrize("checkpoint8", [False, True])
@pytest.mark.parametrize("B,S,vocab", [(2, 128, 1000), (1, 300, 1009)])
def test_loss_and_gradients_against_torch(tm, B, S, vocab, checkpoint8):
    """bf16 model against the torch model in fp32.  The torch model in bf16 is off by its own roundings; the
    library's may be off by twice that, plus, with the 8-bit checkpoint, the error it puts into each
    feed-forward's gradients (0.9% rms of a group's values: 3% of a gradient's norm at most, as in the
    checkpoint's own test)."""
    model = tm.build(vocab, layers=2, checkpoint8=checkpoint8)
    tokens, targets = tm.batch(vocab, B, S, 1)
    ref = copy.deepcopy(model).float()
    loss32, g32 = step(ref, ref.reference, tokens, targets)
    loss16, g16 = step(model, model.reference, tokens, targets)
    loss, g = step(model, model, tokens, targets)
    assert abs(loss - loss32) <= 2 * abs(loss16 - loss32) + 2e-3 * loss32
    for (name, _), a, b, c in zip(model.named_parameters(), g, g16, g32):
        own = ((b - c).norm() / c.norm()).item()
        off = ((a - c).norm() / c.norm()).item()
        assert off <= 2 * own + (0.03 if checkpoint8 else 0.005), (name, off, own)
    assert _ext.device_status() == 0


def test_it_learns(tm):
    losses = tm.main(["--steps", "30", "--layers", "1", "--vocab", "2048", "--batch", "8", "--seq", "256"])
    assert losses[-1] < 0.5 * losses[0]


def test_the_checkpoint_saves_memory(tm):
    """What one step holds at its largest with the feed-forward's activations in 8 and in 16 bits: 6 F bytes
    a row and layer less 2.06 F (F = 4608, 4096 rows, 4 layers: 290 MB), within the allocator's rounding."""
    peak = {}
    for q8 in (True, False):
        model = tm.build(1024, layers=4, checkpoint8=q8)
        tokens, targets = tm.batch(1024, 4, 1024, 0)
        loss = model(tokens, targets)
        del loss
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        base = torch.cuda.memory_allocated()
        loss = model(tokens, targets)
        peak[q8] = torch.cuda.memory_allocated() - base
        del loss, model
    saved = peak[False] - peak[True]
    assert 0.9 * 4 * 4096 * 4608 * (6 - 2.0625) <= saved <= 1.1 * 4 * 4096 * 4608 * (6 - 2.0625)
