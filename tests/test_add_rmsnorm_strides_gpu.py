"""What add_rmsnorm's backward returns where one of its gradients is missing lies in memory as its fake says, whatever
the strides of the gradient that there is: a compiled backward was planned for that."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from add_rmsnorm import add_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"
BF16 = torch.bfloat16


def operands(n=24, d=40):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(*s, generator=g).to(dev, BF16) for s in ((n, d), (n, d), (d,), (n, d))]


def turned(t):
    """The same values, columns first."""
    return t.t().contiguous().t()


@pytest.mark.parametrize("way", ["z alone", "y alone", "both", "neither"])
def test_strides_are_the_fake_ones(way):
    x, res, w, grad = operands()
    y, z, rstd = torch.ops.krsi.add_rmsnorm_fwd(x, res, w, 1e-6)
    gy = turned(grad) if way in ("y alone", "both") else None
    gz = turned(grad) if way in ("z alone", "both") else None
    for zz in (z, turned(z)):
        got = torch.ops.krsi.add_rmsnorm_bwd(gy, gz, zz, w, rstd)
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            fake = [None if t is None else mode.from_tensor(t) for t in (gy, gz, zz, w, rstd)]
            planned = torch.ops.krsi.add_rmsnorm_bwd(*fake)
        assert [t.stride() for t in got] == [t.stride() for t in planned]
        assert [(t.shape, t.dtype) for t in got] == [(t.shape, t.dtype) for t in planned]
        if way == "z alone":
            assert torch.equal(got[0], grad) and not got[1].any()


def test_compiled_with_a_turned_gradient_of_z_alone():
    x, res, w, grad = operands()

    def fn(a, b, c):
        return add_rmsnorm(a, b, c, 1e-6)[1] * 2

    leaves = [[t.clone().requires_grad_(True) for t in (x, res, w)] for _ in range(2)]
    want = torch.autograd.grad(fn(*leaves[0]), leaves[0], turned(grad), allow_unused=True)
    got = torch.autograd.grad(torch.compile(fn, fullgraph=True)(*leaves[1]), leaves[1], turned(grad), allow_unused=True)
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a, b)
    assert got[2] is None or not got[2].any()
