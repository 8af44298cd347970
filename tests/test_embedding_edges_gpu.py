"""The embedding's gradient where its kernels change over: vocabularies and position counts at the limits of
the sort, both sides of the one-launch sum, and runs at the borders of chunks."""
import pytest
import torch

import _ext
from embedding import embedding

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_the_largest_vocabulary_that_is_accepted():
    """The sort's 2^22 groups of 512 tokens: the entry behind the last one is start[2^31], which an int does not
    hold.  600 positions (the sorted path), among them the ends of the vocabulary and of its last group."""
    V = 2 ** 31 - 1025
    last_group = 510 * 2 ** 22 + 2 ** 22 - 1          # the largest token whose low 22 bits are all ones
    tokens = torch.randint(0, V, (600,), generator=torch.Generator().manual_seed(0))
    tokens[:6] = torch.tensor([0, V - 1, last_group, last_group, 2 ** 22 - 1, V - 1])
    g = torch.randint(1, 5, (600, 1), generator=torch.Generator().manual_seed(1)).half()
    table = torch.zeros(1, 1, device=dev, dtype=torch.half).expand(V, 1)   # (the gradient reads its shape alone)
    grad = torch.ops.krsi.embedding_bwd(g.to(dev), tokens.to(dev), table, 1.0, -1)
    ids, at = torch.unique(tokens, return_inverse=True)
    want = torch.zeros(len(ids)).index_add_(0, at, g[:, 0].float())
    assert torch.equal(grad[ids.to(dev), 0].float().cpu(), want)
    assert int(torch.count_nonzero(grad)) == len(ids)
    assert _ext.device_status() == 0


UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def check(grad, tokens, g, V, scale=1.0, skip=None):
    """The gradient against float64.  Additions that a term of a token with `count` positions passes: up to 512
    positions in all, `count` in a row; above, 16 of its chunk, then the m = count / 16 + 2 chunks' sums: in a row up to
    16 of them, else an eighth and 8 more.  Then the scale's product and the result's rounding."""
    t, g = tokens.reshape(-1).cpu().long(), g.reshape(tokens.numel(), -1).cpu().double()
    keep = (t >= 0) & (t < V)
    if skip is not None:
        keep &= t != skip
    t, g = t[keep], g[keep]
    zero = torch.zeros(V, g.shape[1], dtype=torch.float64)
    want, mag = zero.index_add(0, t, g) * scale, zero.index_add(0, t, g.abs()) * abs(scale)
    count = torch.bincount(t, minlength=V)
    m = count // 16 + 2
    adds = count if tokens.numel() <= 512 else 16 + torch.where(m <= 16, m, (m + 7) // 8 + 8)
    bound = (adds + 1)[:, None] * 2.0 ** -24 * mag + 1.01 * UNIT[grad.dtype] * want.abs() + TINY[grad.dtype]
    err = (grad.cpu().double() - want).abs()
    assert torch.all(err <= bound), (err - bound).max()
    assert _ext.device_status() == 0


def ids(n, V, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.exp(torch.rand(n, generator=g) * torch.tensor(float(V)).log()) - 1).long().clamp(0, V - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [400, 511, 512, 513, 2000])
def test_padding_on_both_sides_of_the_one_launch_sum(n, dtype):
    V, d = 50, 96
    tokens = ids(n, V, n)
    tokens[::2] = 7
    g = torch.randn(n, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    for pad in (7, 7 - V):
        t = torch.randn(V, d, generator=torch.Generator().manual_seed(0)).to(dev, dtype).requires_grad_(True)
        out = embedding(tokens.to(dev), t, padding_idx=pad)
        assert torch.equal(out, t[tokens.to(dev)])
        (grad,) = torch.autograd.grad(out, t, g.to(dev))
        check(grad, tokens, g, V, skip=7)
        assert not grad[7].any()
    t = torch.zeros(V, d, device=dev, dtype=dtype, requires_grad=True)     # the padding token alone
    (grad,) = torch.autograd.grad(embedding(torch.full((n,), 7, device=dev), t, padding_idx=7), t, g.to(dev))
    assert not grad.any()


@pytest.mark.parametrize("n", [512, 513, 2000])
@pytest.mark.parametrize("kind", [torch.int64, torch.int32])
def test_tokens_out_of_range_on_both_sides(n, kind):
    V, d = 10, 32
    tokens = ids(n, V, n)
    far = [-1, V, 2 ** 31 - 1, -2 ** 31] + ([2 ** 40, -2 ** 40, 2 ** 32 + 3] if kind is torch.int64 else [])
    for i, bad in enumerate(far):
        tokens[5 + i::37] = bad
    tokens = tokens.to(kind)
    table = torch.randn(V, d, generator=torch.Generator().manual_seed(0))
    g = torch.randn(n, d, generator=torch.Generator().manual_seed(1))
    t = table.to(dev).requires_grad_(True)
    out = embedding(tokens.to(dev), t)
    ok = (tokens >= 0) & (tokens < V)
    assert torch.equal(out.detach().cpu()[ok], table[tokens[ok].long()]) and out.detach().cpu()[~ok].isnan().all()
    (grad,) = torch.autograd.grad(out, t, g.to(dev))
    check(grad, tokens, g, V)
    (none,) = torch.autograd.grad(embedding(torch.full((n,), V, device=dev, dtype=kind), t), t, g.to(dev))
    assert not none.any()


@pytest.mark.parametrize("n", [512, 513, 3000])
@pytest.mark.parametrize("d", [33, 34, 36, 40])
def test_strided_inputs_and_unaligned_rows_on_both_sides(n, d):
    """Token views, transposed gradients and tables that start off the packet alignment, by row width."""
    V = 64
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, V, (n, 3), generator=gen)
    table = torch.randn(V * d + 1, generator=gen).to(dev, torch.bfloat16)[1:].view(V, d).detach().requires_grad_(True)
    g = torch.randn(d, n, generator=gen).to(dev, torch.bfloat16).t()
    out = embedding(tokens.to(dev)[:, 1], table)
    assert torch.equal(out, table[tokens.to(dev)[:, 1]])
    (grad,) = torch.autograd.grad(out, table, g)
    check(grad, tokens[:, 1], g, V)


def test_compiled_above_the_one_launch_sum():
    V, d, n = 100, 64, 2000
    tokens = ids(n, V, 2).to(dev)
    table, g = torch.randn(V, d, device=dev, requires_grad=True), torch.randn(n, d, device=dev)
    fn = torch.compile(lambda t: embedding(tokens, t, 2.0, 3), fullgraph=True)
    a, b = embedding(tokens, table, 2.0, 3), fn(table)
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, table, g)[0], torch.autograd.grad(b, table, g)[0])


@pytest.mark.parametrize("lengths", [
    [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 16, 16, 1, 300, 15, 1, 16],      # chunks of 16 begin and end anywhere
    [16] * 40, [15] * 40, [17] * 40, [256, 257, 255, 1], [272, 273, 271], [16 * 16 + 1, 16 * 17, 16 * 18 - 1, 5],
    [600], [1] * 600, [513], [1, 512], [512, 1]])
def test_runs_by_chunks_of_sixteen(lengths):
    """Runs inside a chunk, over one border and over as many chunks as one warp adds alone (16) and more."""
    V, d = len(lengths) + 3, 24
    tokens = torch.cat([torch.full((k,), i) for i, k in enumerate(lengths)])
    tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(0))]
    g = torch.randn(len(tokens), d, generator=torch.Generator().manual_seed(1))
    t = torch.zeros(V, d, device=dev, requires_grad=True)
    (grad,) = torch.autograd.grad(embedding(tokens.to(dev), t), t, g.to(dev))
    check(grad, tokens, g, V)
    assert not grad[len(lengths):].any()


@pytest.mark.parametrize("n", [32736, 32768, 32769, 65536, 70001])
@pytest.mark.parametrize("V", [3, 4000, 70000])
def test_more_positions_than_a_tile_of_the_sort(n, V):
    """Up to three tiles of 32768 positions, with padding and tokens outside the table; the same bits every time."""
    d = 16
    tokens = ids(n, V, n + V)
    tokens[::5] = V - 1
    tokens[::7] = -3
    tokens[-1] = 0
    g = torch.randn(n, d, generator=torch.Generator().manual_seed(1))
    t = torch.zeros(V, d, device=dev, requires_grad=True)
    for pad in (None, V - 1):
        (grad,) = torch.autograd.grad(embedding(tokens.to(dev), t, 0.5, pad), t, g.to(dev))
        check(grad, tokens, g, V, 0.5, skip=pad)
        (again,) = torch.autograd.grad(embedding(tokens.int().to(dev), t, 0.5, pad), t, g.to(dev))
        assert torch.equal(grad, again)
