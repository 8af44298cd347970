"""The token model's evaluation in 8 bits, row by row: its last hidden rows beside the model's in fp32, and the weights
that it reads."""
import copy
import importlib.util
import math

import pytest
import torch
import torch.nn.functional as F

from conftest import PKG
from linear_q8 import dequantise

pytestmark = pytest.mark.gpu
HEADS, D_KV = 16, 72


@pytest.fixture(scope="module")
def tm():
    spec = importlib.util.spec_from_file_location("krsi_token_model_rows", PKG / "t5_block" / "token_model.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def projections(layer):
    return [m.weight for m in (layer.q, layer.k, layer.v, layer.wi_0, layer.wi_1)]


def rows8(x):
    """The rows of x as 8 bits hold them."""
    top = x.abs().amax(-1, keepdim=True)
    return (x * (448 / top)).to(torch.float8_e4m3fn).float() * (top / 448)


@torch.no_grad()
def hidden(model, tokens, rounded=lambda x: x, plant=lambda i, ws: ws):
    """The definition in fp32, its projections' operands through `rounded` and its weights through `plant`."""
    x = F.embedding(tokens, model.table) * math.sqrt(model.table.shape[1])
    B, S, d = x.shape
    for i, layer in enumerate(model.layers):
        ws = [rounded(w) for w in plant(i, projections(layer))]
        h = rounded(layer.ln1(x))
        q, k, v = (F.linear(h, w).view(B, S, HEADS, D_KV).transpose(1, 2) for w in ws[:3])
        p = torch.softmax(q @ k.transpose(-1, -2) + layer.position_bias(S, x.device), -1)
        x = x + layer.o((p @ v).transpose(1, 2).reshape(B, S, -1))
        h = rounded(layer.ln2(x))
        x = x + layer.wo(F.gelu(F.linear(h, ws[3]), approximate="tanh") * F.linear(h, ws[4]))
    return model.ln(x).reshape(-1, d)


def off(a, b):
    return ((a - b).norm() / b.norm()).item()


def last_rows(tm, monkeypatch, call):
    """What `call` hands to the vocabulary's cross entropy."""
    seen = []
    whole = tm.linear_cross_entropy.linear_cross_entropy

    def spy(h, *a, **kw):
        seen.append(h.detach().float().cpu())
        return whole(h, *a, **kw)

    with monkeypatch.context() as m:
        m.setattr(tm.linear_cross_entropy, "linear_cross_entropy", spy)
        with torch.no_grad():
            call()
    (rows,) = seen
    return rows


@pytest.mark.parametrize("layers", [1, 3])
def test_last_rows(tm, monkeypatch, layers):
    """By norm the rows are off by what the definition with its operands in 8 bits is, and by what the 16-bit model is:
    errors of independent operands add up to the root of their squares, so 5/4 of the one and all of the other is ample.
    One projection with its weight's rows in another order, at any place, is off by more than twice that."""
    model = tm.build(1000, layers=layers, checkpoint8=False)
    tokens, targets = tm.batch(1000, 2, 256, 1)
    weights = model.quantised()
    got8 = last_rows(tm, monkeypatch, lambda: model.evaluate8(tokens, targets, weights))
    got16 = last_rows(tm, monkeypatch, lambda: model(tokens, targets))
    ref, where = copy.deepcopy(model).cpu().float(), tokens.cpu()
    want = hidden(ref, where)
    bound = 1.25 * off(hidden(ref, where, rows8), want) + off(got16, want)
    assert off(got8, want) <= bound
    for at in range(layers):
        for j in range(5):
            def turned(i, ws):
                return [w.roll(1, 0) if (i, k) == (at, j) else w for k, w in enumerate(ws)]
            assert off(hidden(ref, where, plant=turned), want) > 2 * bound


def test_every_weight_is_quantised_in_its_place(tm):
    model = tm.build(515, layers=3, checkpoint8=False)
    pairs = model.quantised()
    assert len(pairs) == 3
    for layer, two in zip(model.layers, pairs):
        ws = projections(layer)
        for (q, scale), part in zip(two, (ws[:3], ws[3:])):
            w = torch.cat(list(part)).detach().double()
            assert q.shape == w.shape and scale.shape == w.shape[:1]
            # half a code: 2^-4 of the value, or 2^-10 of the unit below the least normal code; fp32's rounding of each
            tol = w.abs() * (2 ** -4 + 2 ** -22) + scale.double()[:, None] * 2 ** -9.99
            assert ((dequantise(q, scale).double() - w).abs() <= tol).all()
