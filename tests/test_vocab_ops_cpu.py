"""Host-side contract of the vocabulary operators and the 8-bit GEGLU checkpoint: signatures, operator
schemas, fake (meta) implementations, and the C ABI's argument checks, which return before any device
work.  CPU only."""
import ctypes
import inspect

import pytest
import torch

from conftest import PKG

vp, i64, f32, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(str(PKG / "lib" / "libkrsi_b200.so"))


def test_public_signatures():
    import embedding
    import geglu_q8
    import linear_cross_entropy as ce

    assert list(inspect.signature(embedding.embedding).parameters) == ["tokens", "table", "scale", "padding_idx"]
    assert list(inspect.signature(geglu_q8.geglu_q8).parameters) == ["u"]
    assert list(inspect.signature(geglu_q8.feed_forward_q8).parameters) == ["x2d", "wi", "wo", "res"]
    assert list(inspect.signature(ce.linear_cross_entropy).parameters) == \
        ["x2d", "w", "targets", "scale", "ignore_index", "z_loss", "reduction"]
    for mod in (embedding, geglu_q8, ce):
        assert callable(mod.reference) and callable(mod.selftest)


def test_fake_impls_give_the_shapes():
    import embedding  # noqa: F401

    ops = torch.ops.krsi
    m = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    tok, table = m(3, 5, dtype=torch.long), m(11, 16)
    assert ops.embedding_fwd(tok, table, 1.0, -1).shape == (3, 5, 16)
    assert ops.embedding_bwd(m(3, 5, 16), tok, table, 1.0, -1).shape == (11, 16)
    out, q, ex = ops.geglu_q8_fwd(m(4, 80), True)
    assert out.shape == (4, 40) and q.shape == (4, 80) and q.dtype == torch.int8
    assert ex.shape == (4, 2, 2) and ex.dtype == torch.uint8
    assert [t.shape[0] for t in ops.geglu_q8_fwd(m(4, 80), False)] == [4, 0, 0]
    du, again = ops.geglu_q8_bwd(m(4, 40), q, ex, True)
    assert du.shape == (4, 80) and again.shape == (4, 40)
    x, w, t = m(7, 24), m(100, 24), m(7, dtype=torch.long)
    loss, total, weight, stats, dx, dw = ops.linear_ce_fwd(x, w, t, 1.0, -100, 0.0, 1, True, False)
    assert loss.shape == (7,) and total.shape == () and weight.shape == (1,) and stats.shape == (7, 2) and loss.dtype == torch.float32
    assert dx.shape == (7, 24) and dx.dtype == torch.float32 and dw.shape == (0, 24)
    dx, dw = ops.linear_ce_grad(loss, weight, stats, x, w, t, 1.0, -100, 0.0, False, True)
    assert dx.shape == (0, 24) and dw.shape == (100, 24) and dw.dtype == torch.bfloat16
    assert ops.linear_ce_finish(m(7, 24, dtype=torch.float32), total, weight, 1.0, x).dtype == torch.bfloat16


def test_cpu_tensors_are_rejected():
    from embedding import embedding
    from geglu_q8 import geglu_q8
    from linear_cross_entropy import linear_cross_entropy

    t = torch.zeros(4, dtype=torch.long)
    for call in (lambda: embedding(t, torch.zeros(5, 8)), lambda: geglu_q8(torch.zeros(4, 8)),
                 lambda: linear_cross_entropy(torch.zeros(4, 8).bfloat16(), torch.zeros(5, 8).bfloat16(), t)):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()


def test_embedding_argument_checks(lib):
    fwd, bwd = lib.krsi_embedding_fwd, lib.krsi_embedding_bwd
    assert fwd(vp(0), 64, vp(16), vp(16), i64(4), i64(10), i64(8), f32(1), 0, vp(0)) == 1
    assert fwd(vp(16), 16, vp(16), vp(16), i64(4), i64(10), i64(8), f32(1), 0, vp(0)) == 1
    assert fwd(vp(16), 64, vp(16), vp(16), i64(4), i64(10), i64(8), f32(1), 7, vp(0)) == 1
    assert fwd(vp(16), 64, vp(16), vp(16), i64(-1), i64(10), i64(8), f32(1), 0, vp(0)) == 1
    assert fwd(vp(16), 64, vp(16), vp(16), i64(4), i64(1 << 32), i64(8), f32(1), 0, vp(0)) == 2
    assert fwd(vp(0), 64, vp(0), vp(0), i64(0), i64(10), i64(8), f32(1), 0, vp(0)) == 0
    ws = size(0)
    assert lib.krsi_embedding_bwd_workspace_size(i64(1000), i64(50), i64(64), ctypes.byref(ws)) == 0
    assert ws.value >= 2 * 63 * 64 * 4 + 2 * 4000 + 51 * 4
    args = (i64(1000), i64(50), i64(64), f32(1))
    assert bwd(vp(16), 64, vp(16), vp(16), vp(0), ws, *args, i64(-1), 0, vp(0)) == 4
    assert bwd(vp(16), 64, vp(16), vp(16), vp(16), size(ws.value - 1), *args, i64(-1), 0, vp(0)) == 4
    assert bwd(vp(16), 64, vp(16), vp(16), vp(8), ws, *args, i64(-1), 0, vp(0)) == 3
    assert bwd(vp(16), 64, vp(16), vp(16), vp(16), ws, *args, i64(50), 0, vp(0)) == 1
    assert bwd(vp(16), 64, vp(0), vp(16), vp(16), ws, *args, i64(-1), 0, vp(0)) == 1


def test_geglu_q8_argument_checks(lib):
    fwd, bwd = lib.krsi_geglu_q8_fwd, lib.krsi_geglu_q8_bwd
    assert fwd(vp(0), vp(16), vp(16), vp(16), i64(4), i64(32), 1, vp(0)) == 1
    assert fwd(vp(16), vp(16), vp(16), vp(0), i64(4), i64(32), 1, vp(0)) == 1      # half a checkpoint
    assert fwd(vp(16), vp(16), vp(16), vp(17), i64(4), i64(32), 1, vp(0)) == 3
    assert fwd(vp(16), vp(16), vp(16), vp(16), i64(4), i64(32), 5, vp(0)) == 1
    assert fwd(vp(0), vp(0), vp(0), vp(0), i64(0), i64(32), 1, vp(0)) == 0
    assert bwd(vp(16), vp(0), vp(16), vp(16), vp(0), i64(4), i64(32), 1, vp(0)) == 1
    assert bwd(vp(16), vp(16), vp(16), vp(16), vp(0), i64(-4), i64(32), 1, vp(0)) == 1
    assert bwd(vp(0), vp(0), vp(0), vp(0), vp(0), i64(4), i64(0), 1, vp(0)) == 0


def test_linear_ce_argument_checks(lib):
    def fwd(x=16, w=16, t=16, bits=64, loss=16, n=4, V=10, K=64, dtype=1, stats=0):
        return lib.krsi_linear_ce_fwd(vp(x), vp(w), vp(t), bits, vp(loss), vp(0), vp(0), vp(stats), vp(0), vp(0), vp(256),
                                      size(1 << 30), i64(n), i64(V), i64(K), f32(1), i64(-100), f32(0), 0, dtype, vp(0))

    assert fwd(x=0) == 1 and fwd(loss=0) == 1 and fwd(bits=8) == 1 and fwd(n=-1) == 1 and fwd(V=0) == 1
    assert fwd(dtype=0) == 2 and fwd(K=60) == 2 and fwd(V=1 << 31) == 2
    assert fwd(x=24) == 3 and fwd(stats=12) == 3
    assert fwd(n=0, x=0, w=0, t=0, loss=0) == 0

    def grad(g=16, stats=16, stride=1, dx=16, dw=16, n=4):
        return lib.krsi_linear_ce_grad(vp(16), vp(16), vp(16), 64, vp(g), i64(stride), vp(0), vp(stats), vp(dx), vp(dw),
                                       vp(256), size(1 << 30), i64(n), i64(10), i64(64), f32(1), i64(-100), f32(0), 1,
                                       vp(0))

    assert grad(g=0) == 1 and grad(stats=0) == 1 and grad(stride=2) == 1 and grad(dx=0, dw=0) == 1
    assert grad(stats=12) == 3 and grad(dw=24) == 3 and grad(n=0, dw=0) == 0
    assert lib.krsi_linear_ce_finish(vp(16), vp(0), vp(0), vp(16), i64(12), f32(1), 1, vp(0)) == 2
    assert lib.krsi_linear_ce_finish(vp(0), vp(0), vp(0), vp(16), i64(16), f32(1), 1, vp(0)) == 1
    assert lib.krsi_linear_ce_workspace_size(i64(4), i64(10), i64(64), 3, ctypes.byref(size(0))) == 1


def test_perf_cases_are_well_formed():
    """perf/operators.py: distinct names, plain values, and draws that stay within the listed work."""
    import importlib.util
    import random

    spec = importlib.util.spec_from_file_location("krsi_perf_operators", PKG.parent / "perf" / "operators.py")
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    cases = ops.listed()
    assert len({c["name"] for c in cases}) == len(cases) == 12
    most = max(max(w["bytes"] * 300, w["flops"]) for w in map(ops.work, cases))
    rng = random.Random(0)
    for _ in range(200):
        w = ops.work(ops.draw(rng))
        assert 0 < max(w["bytes"] * 300, w["flops"]) <= most


def test_fake_tensors_pass_the_eager_operators():
    """Shapes of fake CUDA tensors through the public functions, where no kernel can run."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from embedding import embedding
    from geglu_q8 import geglu_q8
    from linear_cross_entropy import linear_cross_entropy

    with FakeTensorMode():
        f = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        t, x, tok = f(50, 64), f(24, 64), f(24, dtype=torch.long)
        for need in (False, True):
            a, b = x.clone().requires_grad_(need), t.clone().requires_grad_(need)
            for y, shape in ((embedding(tok, b), (24, 64)), (geglu_q8(a), (24, 32)),
                             (linear_cross_entropy(a, b, tok), ()),
                             (linear_cross_entropy(a, b, tok, reduction="none"), (24,))):
                assert y.shape == shape and y.device.type == "cuda" and y.requires_grad == need


@pytest.mark.parametrize("vocab", [2, 3, 40, 64, 65, 66, 8192])
def test_token_model_batches_stay_in_the_vocabulary(vocab):
    """The synthetic sequences of any vocabulary: tokens and targets below its mask token, which stands for the
    masked positions; the step from token to token holds.  From 65 on the sequences are the same ones."""
    import importlib.util

    spec = importlib.util.spec_from_file_location("krsi_token_model_cpu", PKG / "t5_block" / "token_model.py")
    tm = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(tm)
    tokens, targets = tm.batch(vocab, 4, 100, 3, device="cpu")
    masked = targets != tm.IGNORE
    assert masked.any() and torch.equal(masked, tokens == vocab - 1)
    text = torch.where(masked, targets, tokens)
    used = min(64, vocab - 1)
    assert text.min() >= 0 and text.max() < vocab - 1
    assert torch.equal(text[:, 1:], (5 * text[:, :-1] + 3) % used)
    with pytest.raises(ValueError, match="mask token"):
        tm.batch(1, 4, 100, 3, device="cpu")


def test_linear_ce_workspace_modes(lib):
    """Kinds 0 to 2, and with gradients at most one of the two flags; refused before the device is asked."""
    for mode in (-1, 3, 4, 8, 7, 11, 13, 14, 16, 17):
        assert lib.krsi_linear_ce_workspace_size(i64(4), i64(10), i64(64), mode, ctypes.byref(size(0))) == 1, mode
    for mode in (0, 1, 2, 5, 6, 9, 10):
        assert lib.krsi_linear_ce_workspace_size(i64(4), i64(10), i64(64), mode, ctypes.byref(size(0))) != 1, mode
