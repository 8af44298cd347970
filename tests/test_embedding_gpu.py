"""The embedding lookup and its table gradient (B200) against the definition in float64: types, odd
sizes, token types and orders, empty and heavy tokens, refusals, and the sorted sum's determinism."""
import pytest
import torch

import _ext
from embedding import embedding, reference

pytestmark = pytest.mark.gpu
dev = "cuda"
# one rounding of the result's type, relative to it: 2^-p for a significand of p bits (24, 8, 11)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ids_of(n, V, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "zipf":
        return (torch.exp(torch.rand(n, generator=g) * torch.tensor(float(V)).log()) - 1).long().clamp(0, V - 1)
    if kind == "one":
        return torch.full((n,), V // 2)
    if kind == "last":
        return torch.full((n,), V - 1)
    return torch.randint(0, V, (n,), generator=g)


def exact_grad(tokens, g, V, scale, skip=None):
    """(sum, sum of magnitudes) per table entry in float64."""
    t, g = tokens.reshape(-1), g.reshape(tokens.numel(), -1).double()
    keep = (t >= 0) & (t < V)
    if skip is not None:
        keep &= t != skip
    t, g = t[keep].long(), g[keep]
    out, mag = torch.zeros(V, g.shape[1], dtype=torch.float64), torch.zeros(V, g.shape[1], dtype=torch.float64)
    return out.index_add_(0, t, g) * scale, mag.index_add_(0, t, g.abs()) * abs(scale)


def check_grad(got, tokens, g, V, scale, skip=None):
    want, mag = exact_grad(tokens, g, V, scale, skip)
    count = max(1, int(torch.bincount(tokens.reshape(-1).clamp(0, V - 1).long()).max()) if tokens.numel() else 1)
    # fp32 sum of `count` terms in chunks: each term passes fewer than 64 + count / 32 additions, then the
    # scale's product; then the result's rounding (and the smallest subnormal's half)
    terms = min(count, 64 + count // 32) + 2
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[got.dtype]
    bound = terms * 2.0 ** -24 * mag + UNIT[got.dtype] * want.abs() * 1.01 + tiny
    err = (got.cpu().double() - want).abs()
    assert torch.all(err <= bound), (err - bound).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 1000, 64), (33, 7, 3), (257, 1009, 250), (1000, 5, 72),
                                   (2048, 32768, 1152), (777, 151, 1151), (64, 300, 4100), (31, 40, 2047)])
def test_lookup_and_gradient(n, V, d, dtype):
    tokens = ids_of(n, V, n + d)
    gen = torch.Generator().manual_seed(d)
    table = torch.randn(V, d, generator=gen).to(dtype)
    g = torch.randn(n, d, generator=gen).to(dtype)
    t = table.to(dev).requires_grad_(True)
    out = embedding(tokens.to(dev), t, scale=0.37)
    want = (table[tokens].double() * torch.tensor(0.37).double()).to(dtype)   # 0.37 as the kernel's fp32
    assert out.dtype == dtype and torch.equal(out.detach().cpu(), (table[tokens].float() * 0.37).to(dtype)), want
    (grad,) = torch.autograd.grad(out, t, g.to(dev))
    check_grad(grad, tokens, g, V, float(torch.tensor(0.37)))
    assert _ext.device_status() == 0


@pytest.mark.parametrize("kind", ["one", "last", "uniform"])
@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 1025, 20000])
def test_runs_that_cross_chunks(n, kind):
    """All positions one token, or spread: runs inside a chunk, across one boundary and across hundreds."""
    V, d = 37, 40
    tokens = ids_of(n, V, 3, kind)
    g = torch.randn(n, d, generator=torch.Generator().manual_seed(n))
    t = torch.zeros(V, d, device=dev, requires_grad=True)
    (grad,) = torch.autograd.grad(embedding(tokens.to(dev), t), t, g.to(dev))
    check_grad(grad, tokens, g, V, 1.0)


def test_alternating_runs_of_every_length():
    lengths = [1, 2, 31, 32, 33, 63, 64, 65, 100, 1, 1, 200, 32, 32, 1]
    V, d = len(lengths), 24
    tokens = torch.cat([torch.full((n,), i) for i, n in enumerate(lengths)])
    tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(0))]
    g = torch.randn(len(tokens), d, generator=torch.Generator().manual_seed(1))
    t = torch.zeros(V + 3, d, device=dev, requires_grad=True)     # the last three tokens never occur
    (grad,) = torch.autograd.grad(embedding(tokens.to(dev), t), t, g.to(dev))
    check_grad(grad, tokens, g, V + 3, 1.0)
    assert torch.equal(grad[V:], torch.zeros(3, d, device=dev))


def test_large_vocabulary_and_int32_tokens():
    """A vocabulary above 1024 tokens per block of the sort, and both token types."""
    V, d, n = 300_001, 16, 3000
    tokens = ids_of(n, V, 5, "uniform")
    tokens[:3] = torch.tensor([V - 1, 0, V - 1])
    g = torch.randn(n, d, generator=torch.Generator().manual_seed(2))
    grads = []
    for tt in (tokens, tokens.int()):
        t = torch.zeros(V, d, device=dev, requires_grad=True)
        out = embedding(tt.to(dev), t)
        grads.append(torch.autograd.grad(out, t, g.to(dev))[0])
    check_grad(grads[0], tokens, g, V, 1.0)
    assert torch.equal(grads[0], grads[1])


def test_padding_and_shapes():
    V, d = 50, 96
    tokens = ids_of(400, V, 1).reshape(4, 100)
    tokens[:, ::2] = 7
    table = torch.randn(V, d, generator=torch.Generator().manual_seed(0))
    g = torch.randn(4, 100, d, generator=torch.Generator().manual_seed(1))
    for pad in (7, 7 - V):
        t = table.to(dev).requires_grad_(True)
        out = embedding(tokens.to(dev), t, padding_idx=pad)
        assert out.shape == (4, 100, d) and torch.equal(out.detach().cpu(), table[tokens])
        (grad,) = torch.autograd.grad(out, t, g.to(dev))
        check_grad(grad, tokens, g, V, 1.0, skip=7)
        assert not grad[7].any()


def test_strided_inputs_and_unaligned_rows():
    """Tokens and gradients that are views, a table whose rows start off the packet alignment."""
    V, d, n = 64, 33, 200
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, V, (n, 3), generator=gen)
    store = torch.randn(V * d + 1, generator=gen).to(dev, torch.bfloat16)
    table = store[1:].view(V, d)
    g = torch.randn(d, n, generator=gen).to(dev, torch.bfloat16).t()
    t = table.detach().requires_grad_(True)
    out = embedding(tokens.to(dev)[:, 1], t)
    assert torch.equal(out, table[tokens.to(dev)[:, 1]])
    (grad,) = torch.autograd.grad(out, t, g)
    check_grad(grad, tokens[:, 1], g.cpu(), V, 1.0)


def test_tokens_out_of_range_are_nan_and_get_no_gradient():
    V, d = 10, 32
    tokens = torch.tensor([3, -1, V, 2, -2 ** 40, 2 ** 40, 9])
    table = torch.randn(V, d, generator=torch.Generator().manual_seed(0))
    t = table.to(dev).requires_grad_(True)
    out = embedding(tokens.to(dev), t)
    ok = (tokens >= 0) & (tokens < V)
    assert torch.equal(out.detach().cpu()[ok], table[tokens[ok]]) and out.detach().cpu()[~ok].isnan().all()
    g = torch.randn(len(tokens), d, generator=torch.Generator().manual_seed(1))
    (grad,) = torch.autograd.grad(out, t, g.to(dev))
    check_grad(grad, tokens, g, V, 1.0)


def test_empty():
    for shape in ((0,), (3, 0)):
        t = torch.randn(20, 8, device=dev, requires_grad=True)
        out = embedding(torch.empty(shape, dtype=torch.long, device=dev), t)
        assert out.shape == (*shape, 8)
        (grad,) = torch.autograd.grad(out, t, torch.empty_like(out))
        assert torch.equal(grad, torch.zeros_like(grad))


def test_special_values_pass():
    table = torch.tensor([[float("inf"), float("nan"), -0.0, 1e-40]], device=dev)
    assert torch.equal(embedding(torch.zeros(1, dtype=torch.long, device=dev), table).view(torch.int32),
                       table.view(torch.int32))
    g = torch.tensor([[float("inf"), float("nan"), 1.0, 2.0]] * 2, device=dev)
    t = torch.zeros(3, 4, device=dev, requires_grad=True)
    (grad,) = torch.autograd.grad(embedding(torch.tensor([1, 1], device=dev), t), t, g)
    assert grad[1, 0] == float("inf") and grad[1, 1].isnan() and grad[1, 2:].tolist() == [2.0, 4.0]
    assert not grad[0].any() and not grad[2].any()


def test_same_bits_every_time_and_on_another_stream():
    V, d, n = 1000, 256, 30000
    tokens = ids_of(n, V, 9).to(dev)
    g = torch.randn(n, d, device=dev, dtype=torch.bfloat16)
    table = torch.zeros(V, d, device=dev, dtype=torch.bfloat16)
    a = torch.ops.krsi.embedding_bwd(g, tokens, table, 1.0, -1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = torch.ops.krsi.embedding_bwd(g, tokens, table, 1.0, -1)
    s.synchronize()
    assert torch.equal(a, b)


def test_gradient_against_differences():
    """d sum(w * out) / d table by a finite step: the op is linear in the table, so the quotient is exact
    up to fp32 rounding of the two sums (about 400 terms of size 1 around a step of 1: 1e-4)."""
    V, d = 6, 8
    tokens = torch.tensor([0, 3, 3, 5, 0, 0], device=dev)
    table = torch.randn(V, d, device=dev, requires_grad=True)
    w = torch.randn(6, d, device=dev)
    (grad,) = torch.autograd.grad(embedding(tokens, table, 1.5), table, w)
    for v, c in ((0, 1), (3, 4), (5, 7), (1, 0)):
        step = torch.zeros_like(table)
        step[v, c] = 1.0
        hi = (embedding(tokens, table.detach() + step, 1.5) * w).sum()
        lo = (embedding(tokens, table.detach() - step, 1.5) * w).sum()
        assert abs(((hi - lo) / 2 - grad[v, c]).item()) < 1e-4


def test_compiled_matches_eager():
    V, d = 100, 64
    tokens = ids_of(300, V, 2).to(dev)
    table = torch.randn(V, d, device=dev, requires_grad=True)
    g = torch.randn(300, d, device=dev)
    fn = torch.compile(lambda t: embedding(tokens, t, 2.0, 3), fullgraph=True)
    a, b = embedding(tokens, table, 2.0, 3), fn(table)
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, table, g)[0], torch.autograd.grad(b, table, g)[0])


def test_matches_the_torch_expression():
    tokens = ids_of(500, 90, 4).to(dev)
    t1 = torch.randn(90, 48, device=dev, requires_grad=True)
    t2 = t1.detach().clone().requires_grad_(True)
    a, b = embedding(tokens, t1, 3.0, 0), reference(tokens, t2, 3.0, 0)
    assert torch.equal(a, b)
    g = torch.randn_like(a)
    ga, gb = torch.autograd.grad(a, t1, g)[0], torch.autograd.grad(b, t2, g)[0]
    assert torch.allclose(ga, gb, rtol=1e-4, atol=1e-4)


def test_refusals():
    table = torch.randn(10, 16, device=dev)
    tokens = torch.zeros(4, dtype=torch.long, device=dev)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        embedding(tokens.float(), table)
    with pytest.raises(RuntimeError, match=r"\[V, d\]"):
        embedding(tokens, table[0])
    with pytest.raises(RuntimeError, match="dtype"):
        embedding(tokens, table.double())
    with pytest.raises((RuntimeError, NotImplementedError)):
        embedding(tokens.cpu(), table)
    for pad in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding(tokens, table, padding_idx=pad)
    with pytest.raises(RuntimeError, match="g must be"):
        torch.ops.krsi.embedding_bwd(torch.zeros(3, 16, device=dev), tokens, table, 1.0, -1)
