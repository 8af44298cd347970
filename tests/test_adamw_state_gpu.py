"""AdamW's state dictionary when it comes back from another device."""
import pytest
import torch

from adamw import AdamW

pytestmark = pytest.mark.gpu
dev = "cuda"


def params(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dev, torch.bfloat16).requires_grad_(True) for s in ((70, 90), (33,))]


def steps(ps, opt, first, count):
    for k in range(first, first + count):
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * k + i)).to(dev, p.dtype)
        opt.step()


def on_cpu(tree):
    if isinstance(tree, torch.Tensor):
        return tree.cpu()
    if isinstance(tree, dict):
        return {k: on_cpu(v) for k, v in tree.items()}
    return [on_cpu(v) for v in tree] if isinstance(tree, list) else tree


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("tensor_lr", [False, True])
def test_loaded_from_a_checkpoint_on_the_cpu(bits, tensor_lr):
    """The states, the step and a tensor lr return to the parameters' device; training goes on with the same bits, also
    captured into a graph at once."""
    def make(ps):
        lr = torch.full((), 1e-2, device=dev) if tensor_lr else 1e-2
        return AdamW([{"params": ps[:1]}, {"params": ps[1:], "weight_decay": 0.0}], lr=lr, bits=bits, master=True,
                     min_8bit_size=100)

    whole, ps = params(), params()
    opt_whole, opt = make(whole), make(ps)
    steps(whole, opt_whole, 0, 5)
    steps(ps, opt, 0, 3)
    saved = on_cpu(opt.state_dict())
    assert not saved["param_groups"][0]["step"].is_cuda
    again = params(1)
    with torch.no_grad():
        for p, q in zip(again, ps):
            p.copy_(q)
    opt2 = make(again)
    opt2.load_state_dict(saved)
    for group in opt2.param_groups:
        assert group["step"].is_cuda and group["step"].item() == 3
        assert not tensor_lr or (group["lr"].is_cuda and group["lr"].dtype == torch.float32)
    steps(again, opt2, 3, 1)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        opt2.step()
    for i, p in enumerate(again):   # the gradients of the fifth step, where the graph reads them
        p.grad.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(40 + i)))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    assert [g["step"].item() for g in opt2.param_groups] == [5, 5]
