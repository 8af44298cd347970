"""What the 8-bit GEGLU checkpoint (B200) writes and keeps: in eager and compiled calls, with and without a
backward to come."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from geglu_q8 import feed_forward_q8, geglu_q8

pytestmark = pytest.mark.gpu
dev = "cuda"


class Kept(TorchDispatchMode):
    """The `keep` of each krsi::geglu_q8_fwd that passes."""

    def __init__(self):
        super().__init__()
        self.calls = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func is torch.ops.krsi.geglu_q8_fwd.default:
            self.calls.append(args[1])
        return func(*args, **(kwargs or {}))


def operands(rows=64, d=64, F=96, which=(True,) * 4):
    g = torch.Generator().manual_seed(0)
    make = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dev, torch.bfloat16)  # noqa: E731
    return [t.requires_grad_(w) for t, w in zip((make(rows, d), make(2 * F, d), make(d, F), make(rows, d)), which)]


def kept(fn, *args):
    with Kept() as mode:
        out = fn(*args)
    assert len(mode.calls) == 1
    return mode.calls[0], out


@pytest.mark.parametrize("compiled", [False, True])
def test_no_checkpoint_without_a_backward(compiled):
    """The mode sees what the compiled graph runs, since the operator is opaque to the compiler."""
    torch._dynamo.reset()
    wrap = (lambda f: torch.compile(f, fullgraph=True, backend="aot_eager")) if compiled else (lambda f: f)
    gg, ff = wrap(geglu_q8), wrap(feed_forward_q8)
    x, wi, wo, res = operands()
    u = (x @ wi.t()).detach()
    keep, out = kept(gg, u.clone().requires_grad_(True))
    assert keep
    again, plain = kept(gg, u)
    assert not again and torch.equal(out, plain)
    keep, out = kept(ff, x, wi, wo, res)
    assert keep
    with torch.no_grad():
        keep, plain = kept(ff, x, wi, wo, res)
    assert not keep and torch.equal(out, plain)
    keep, plain = kept(ff, *[t.detach() for t in (x, wi, wo, res)])
    assert not keep and torch.equal(out, plain)


@pytest.mark.parametrize("which", [(False, False, False, True), (True, False, False, False), (False, True, False, True),
                                   (False, False, True, False)])
def test_only_the_gradients_that_are_asked_for(which):
    """Some inputs' gradients alone: the same bits as among all of them; res's alone needs no checkpoint."""
    full = operands()
    want = torch.autograd.grad(feed_forward_q8(*full), full, torch.ones(64, 64, device=dev, dtype=torch.bfloat16))
    some = operands(which=which)
    keep, out = kept(feed_forward_q8, *some)
    assert keep == any(which[:3])
    need = [t for t in some if t.requires_grad]
    got = torch.autograd.grad(out, need, torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(got, [w for w, n in zip(want, which) if n]))


@pytest.mark.parametrize("residual", [True, False])
def test_compiled_feed_forward_keeps_the_checkpoint_alone(residual):
    """What is held between forward and backward besides the output: 2.0625 F bytes a row, compiled and not (the
    rows' count makes the allocator's 512-byte rounding small); and the same bits of outputs and gradients."""
    torch._dynamo.reset()
    rows, d, F = 4096, 128, 1024
    args = operands(rows, d, F)[:4 if residual else 3]
    gy = torch.randn(rows, d, device=dev).bfloat16()
    results = []
    for fn in (feed_forward_q8, torch.compile(feed_forward_q8, fullgraph=True)):
        fn(*args)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = fn(*args)
        held = torch.cuda.memory_allocated() - before - out.numel() * 2
        assert abs(held - 2.0625 * F * rows) <= 0.02 * F * rows, held / (F * rows)
        results.append((out, *torch.autograd.grad(out, args, gy)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
