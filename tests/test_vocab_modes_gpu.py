"""The embedding, the vocabulary cross entropy and the 8-bit GEGLU under torch's own modes: forward-mode
differentiation, dispatch modes, fake tensors, in-place changes and gradients of gradients."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from embedding import embedding
from geglu_q8 import feed_forward_q8, geglu_q8
from linear_cross_entropy import KEEP_ROWS, linear_cross_entropy

pytestmark = pytest.mark.gpu
dev = "cuda"
N, V, K = 24, 50, 64
NAMES = ["embedding", "cross entropy", "cross entropy rows", "geglu", "feed forward"]


def calls():
    """(name, function of float tensors, those tensors) of every public function."""
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g).to(dev, torch.bfloat16)  # noqa: E731
    tokens = torch.randint(0, V, (N,), generator=g).to(dev)
    return {   # (of NAMES)
        "embedding": (lambda t: embedding(tokens, t, 0.5), [rand(V, K)]),
        "cross entropy": (lambda x, w: linear_cross_entropy(x, w, tokens), [rand(N, K), rand(V, K)]),
        "cross entropy rows": (lambda x, w: linear_cross_entropy(x, w, tokens, reduction="none"),
                               [rand(N, K), rand(V, K)]),
        "geglu": (geglu_q8, [rand(N, 2 * K)]),
        "feed forward": (feed_forward_q8, [rand(N, K), rand(2 * V, K), rand(K, V), rand(N, K)]),
    }


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, requires_grad):
    """A tangent that an operator cannot carry is an error, not a derivative of zero; each input in turn."""
    fn, args = calls()[name]
    for i in range(len(args)):
        with fwd_ad.dual_level():
            inputs = [a.clone().requires_grad_(requires_grad) for a in args]
            inputs[i] = fwd_ad.make_dual(inputs[i], torch.ones_like(inputs[i]))
            with pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
                fn(*inputs)
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
                fn(*inputs)
    if name != "feed forward":   # (torch.func refuses Python autograd functions of the old style altogether)
        with pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
            torch.func.jvp(fn, tuple(args), tuple(torch.ones_like(a) for a in args))
    fn(*args)   # and plain tensors still pass


OPS = {   # the operators of a step of each function, forward and backward
    "embedding": {"embedding_fwd", "embedding_grad"},
    "cross entropy": {"linear_ce_fwd", "linear_ce_grad"},
    "cross entropy rows": {"linear_ce_fwd", "linear_ce_grad"},
    "geglu": {"geglu_q8_fwd", "geglu_q8_bwd"},
    "feed forward": {"geglu_q8_fwd", "geglu_q8_bwd"},
}


class Seen(TorchDispatchMode):
    """The krsi operators that pass, and the calls themselves."""

    def __init__(self):
        super().__init__()
        self.ops = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "krsi":
            self.ops.add(func._opname)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", NAMES)
def test_a_dispatch_mode_sees_the_operators(name):
    fn, args = calls()[name]
    args = [a.requires_grad_(True) for a in args]
    with Seen() as seen:
        out = fn(*args)
        torch.autograd.grad(out, args, torch.ones_like(out))
    assert OPS[name] <= seen.ops, seen.ops
    for mode in (torch.no_grad, torch.inference_mode):
        with Seen() as seen, mode():
            plain = fn(*args)
        assert len(seen.ops) == 1 and torch.equal(plain, out), seen.ops


@pytest.mark.parametrize("name", NAMES)
def test_fake_tensors_get_shapes(name):
    """Under a fake-tensor mode no kernel runs; outputs and gradients have the real ones' shapes and types."""
    fn, args = calls()[name]
    args = [a.requires_grad_(True) for a in args]
    out = fn(*args)
    grads = torch.autograd.grad(out, args, torch.ones_like(out))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:   # (the integer inputs are real)
        fakes = [mode.from_tensor(a.detach()).requires_grad_(True) for a in args]
        fake = fn(*fakes)
        fake_grads = torch.autograd.grad(fake, fakes, torch.ones_like(fake))
        with torch.inference_mode():
            again = fn(*[f.detach() for f in fakes])
    for got, want in zip((fake, again, *fake_grads), (out, out, *grads)):
        assert got.shape == want.shape and got.dtype == want.dtype and got.device == want.device


def test_a_table_changed_in_place_before_the_backward():
    """As with torch's embedding: the gradient needs the table's shape alone, and the table is not kept alive."""
    tokens = torch.randint(0, V, (600,), device=dev)
    g = torch.randn(600, K, device=dev)
    for fn in (embedding, torch.compile(embedding, fullgraph=True)):
        table = torch.randn(V, K, device=dev, requires_grad=True)
        (want,) = torch.autograd.grad(fn(tokens, table), table, g)
        out = fn(tokens, table)
        with torch.no_grad():
            table.mul_(0.5)
        (got,) = torch.autograd.grad(out, table, g)
        assert torch.equal(got, want)


def test_embedding_grad_refusals():
    op = torch.ops.krsi.embedding_grad
    tokens, g = torch.zeros(4, dtype=torch.long, device=dev), torch.zeros(4, 8, device=dev)
    assert op(g, tokens, 5, 1.0, -1).shape == (5, 8)
    for bad in (lambda: op(g[:3], tokens, 5, 1.0, -1), lambda: op(g, tokens, 5, 1.0, 5), lambda: op(g, tokens, 0, 1.0, -1),
                lambda: op(g, tokens.float(), 5, 1.0, -1), lambda: op(g.double(), tokens, 5, 1.0, -1)):
        with pytest.raises(RuntimeError):
            bad()


def test_operands_changed_in_place_after_their_gradients_were_formed():
    """From KEEP_ROWS rows on the forward of a reduced loss forms both gradients; what they were formed from may
    then change or be freed.  (Gradients formed later need their operands and refuse a change.)"""
    rows = KEEP_ROWS
    t = torch.randint(0, V, (rows,), device=dev)
    x0, w0 = torch.randn(rows, K, device=dev).bfloat16(), torch.randn(V, K, device=dev).bfloat16()
    for fn in (linear_cross_entropy, torch.compile(linear_cross_entropy, fullgraph=True)):
        x, w = x0.clone().requires_grad_(True), w0.clone().requires_grad_(True)
        want = torch.autograd.grad(fn(x, w, t), (x, w))
        loss = fn(x, w, t)
        with torch.no_grad():
            w.mul_(0.5)
            x.zero_()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), want))
    x, w = x0[:100].clone().requires_grad_(True), w0.clone().requires_grad_(True)
    loss = linear_cross_entropy(x, w, t[:100])
    with torch.no_grad():
        w.mul_(0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, x)


@pytest.mark.parametrize("name", NAMES)
def test_a_gradient_of_the_gradient_is_refused(name):
    fn, args = calls()[name]
    args = [a.requires_grad_(True) for a in args]
    out = fn(*args)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out, args, torch.ones_like(out), create_graph=True)
