"""The embedding, the vocabulary cross entropy and the 8-bit GEGLU under torch's own modes: forward-mode
differentiation, dispatch modes, fake tensors, in-place changes and gradients of gradients."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from embedding import embedding
from geglu_q8 import feed_forward_q8, geglu_q8
from linear_cross_entropy import linear_cross_entropy

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
