"""The token model on the residual norms, the 8-bit projections and the library's AdamW together."""
import copy
import importlib.util

import pytest
import torch

import _ext
from conftest import PKG
from linear_q8 import dequantise, quantise

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tm():
    spec = importlib.util.spec_from_file_location("krsi_token_model_q8", PKG / "t5_block" / "token_model.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def step(model, fn, tokens, targets):
    loss = fn(tokens, targets)
    return loss.detach(), [p.float() for p in torch.autograd.grad(loss, list(model.parameters()))]


@pytest.mark.parametrize("B,S,vocab", [(2, 128, 1000), (1, 300, 1009)])
def test_junctions_against_torch(tm, B, S, vocab):
    """The bf16 model whose residual sums are inside the norms, against the torch model in fp32: off by at most twice
    what the torch model in bf16 is, plus half a percent (its roundings are fewer)."""
    model = tm.build(vocab, layers=2, checkpoint8=False, junctions=True)
    tokens, targets = tm.batch(vocab, B, S, 1)
    ref = copy.deepcopy(model).float()
    loss32, g32 = step(ref, ref.reference, tokens, targets)
    loss16, g16 = step(model, model.reference, tokens, targets)
    loss, g = step(model, model, tokens, targets)
    assert abs(loss - loss32) <= 2 * abs(loss16 - loss32) + 2e-3 * loss32
    for (name, _), a, b, c in zip(model.named_parameters(), g, g16, g32):
        own, off = ((b - c).norm() / c.norm()).item(), ((a - c).norm() / c.norm()).item()
        assert off <= 2 * own + 0.005, (name, off, own)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("layers", [0, 1, 3])
def test_evaluation_in_8_bits(tm, layers):
    """The loss with the projections behind the norms in 8 bits, beside the 16-bit one.  A code is off by 2^-4 at
    most (2.6% rms), so the last norm's output by some 10% after three layers; logits have a spread of about one, so
    a row's loss moves by about 0.1 at random, the mean over 38 targets or more by 0.1 / 38^0.5: six of that."""
    model = tm.build(1000, layers=layers, checkpoint8=False)
    tokens, targets = tm.batch(1000, 2, 256, 1)
    assert (targets != tm.IGNORE).sum() >= 38
    weights = model.quantised()
    with torch.no_grad():
        loss = model(tokens, targets)
    loss8 = model.evaluate8(tokens, targets, weights)
    assert abs(loss8 - loss) <= 0.1
    assert not loss8.requires_grad
    if layers == 0:
        assert torch.equal(loss, loss8)
    for (wqkv, wscale), _ in weights:   # the weights' rows, quantised once
        layer = torch.cat([model.layers[0].q.weight, model.layers[0].k.weight, model.layers[0].v.weight])
        q, s = quantise(layer.detach())
        assert torch.equal(dequantise(q, s), dequantise(wqkv, wscale))
        break


@pytest.mark.parametrize("name", ["adamw", "adamw8"])
def test_training_with_the_library_optimizer_runs(tm, name):
    """Steps of the whole model: every parameter moves and stays finite, in as many steps as were taken."""
    model = tm.build(515, layers=1, junctions=True)
    old = [p.detach().clone() for p in model.parameters()]
    opt = tm.optimizer(name, model.parameters(), 1e-2)
    for k in range(3):
        loss = model(*tm.batch(515, 2, 96, k))
        loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
    assert torch.isfinite(loss) and opt.param_groups[0]["step"].item() == 3
    for p, o in zip(model.parameters(), old):
        assert torch.isfinite(p).all() and not torch.equal(p, o)
    state = opt.state[model.table]["exp_avg"]
    assert state.dtype == (torch.float8_e4m3fn if name == "adamw8" else torch.float32)


def test_command_line(tm, capsys):
    tm.main(["--steps", "4", "--layers", "1", "--vocab", "300", "--batch", "2", "--seq", "128", "--optimizer", "adamw8",
             "--junctions"])
    assert "in 8 bits" in capsys.readouterr().out
