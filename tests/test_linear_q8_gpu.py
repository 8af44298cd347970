"""linear_q8 and quantise against float64, at sizes that end inside every tile.

Tolerance: a product of two e4m3 is exact in fp32; the fp32 sum of K of them is off by at most K 2^-23 of the sum of
magnitudes (a tensor core may drop bits instead of rounding them), three fp32 products by 2^-24 each, the result by
half a step of its type."""
import pytest
import torch

import _ext
from linear_q8 import dequantise, linear_q8, quantise

pytestmark = pytest.mark.gpu
dev = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def operands(rows, K, M, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, K, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dev)
    w = (torch.randn(M, K, generator=g) * K ** -0.5).to(dev)
    return (*quantise(x), *quantise(w))


def check(out, q, scale, wq, wscale):
    a, b = dequantise(q, scale).double(), dequantise(wq, wscale).double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    half = torch.finfo(out.dtype).eps / 2
    low = torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    tol = half * want.abs() + (q.shape[1] * 2 ** -23 + 4 * 2 ** -24) * (1 + half) * size + low
    assert ((out.double() - want).abs() <= tol).all()


# one row, one column, K inside one swizzle row and across many blocks (the ring wraps), rows and columns just below,
# at and above the tiles of either kernel, odd ones, and more tiles than the grid has blocks
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,K,M", [
    (1, 1, 1), (1, 16, 8), (3, 33, 5), (16, 1152, 1000), (127, 128, 64), (128, 129, 65), (128, 2000, 10300),
    (129, 127, 255), (256, 1152, 256), (257, 1000, 257), (300, 100, 2743), (1000, 4608, 513), (2500, 200, 4104)])
def test_against_float64(rows, K, M, dtype):
    ops = operands(rows, K, M)
    out = linear_q8(*ops, dtype)
    assert out.shape == (rows, M) and out.dtype == dtype
    check(out, *ops)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [-1, 0, 2])
@pytest.mark.parametrize("rows,K,M0", [(260, 642, 2400), (257, 145, 3624), (257, 1061, 4768), (523, 86, 3888),
                                       (521, 902, 4640), (781, 1033, 4056)])
def test_widths_of_tiles(rows, K, M0, M, dtype):
    """On 148 SMs: fp32 tiles of 96 to 256 columns, 16-bit ones of 128 to 256, uneven parts among them; rows of out on
    16, 8 or 4 bytes and less."""
    ops = operands(rows, K, M0 + M)
    check(linear_q8(*ops, dtype), *ops)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("rows,K,M,dtype", [(3748, 2608, 4768, F32), (3748, 300, 4768, F32), (3000, 256, 4704, F32),
                                            (3748, 512, 4800, BF16), (3748, 130, 4736, F16), (100, 2000, 20488, F32)])
def test_columns_end_inside_a_tile(rows, K, M, dtype):
    """A tile's last boxes may lie past M: what is written to shared memory for them must not reach the boxes before,
    which are still on their way to memory."""
    g = torch.Generator(device=dev).manual_seed(5)
    q, wq = (torch.randint(-3, 4, (n, K), generator=g, device=dev).to(torch.float8_e4m3fn) for n in (rows, M))
    one = lambda n: torch.ones(n, device=dev)  # noqa: E731
    want = (q.double() @ wq.double().t()).to(dtype)
    for _ in range(3):
        assert torch.equal(linear_q8(q, one(rows), wq, one(M), dtype), want)


@pytest.mark.parametrize("rows", [64, 400])
def test_whole_numbers_are_exact(rows):
    """Small whole numbers have exact products and sums: every element, whatever the order."""
    g = torch.Generator().manual_seed(3)
    q = torch.randint(-8, 9, (rows, 272), generator=g).to(dev).to(torch.float8_e4m3fn)
    wq = torch.randint(-8, 9, (520, 272), generator=g).to(dev).to(torch.float8_e4m3fn)
    one = lambda n: torch.ones(n, device=dev)  # noqa: E731
    out = linear_q8(q, one(rows), wq, one(520), F32)
    assert torch.equal(out.double(), q.double() @ wq.double().t())
    scale = torch.exp2(torch.arange(rows, device=dev) % 7 - 3.0)
    wscale = torch.exp2(torch.arange(520, device=dev) % 5 - 2.0)
    assert torch.equal(linear_q8(q, scale, wq, wscale, F32), out * scale[:, None] * wscale)


def test_layouts_streams_and_repetition():
    """Rows off 16 bytes, transposed, expanded and padded ones; another stream; the same bits every time."""
    q, scale, wq, wscale = operands(200, 100, 120)
    want = linear_q8(q, scale, wq, wscale, F32)
    assert torch.equal(want, linear_q8(q.contiguous(), scale, wq.contiguous(), wscale, F32))
    as8 = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    turned = as8(q).t().contiguous().t().view(torch.float8_e4m3fn)
    assert turned.stride() == (1, 200) and torch.equal(want, linear_q8(turned, scale, wq, wscale, F32))
    wide = torch.zeros(200, 144, dtype=torch.uint8, device=dev)
    wide[:, 16:116] = as8(q)
    assert torch.equal(want, linear_q8(wide.view(torch.float8_e4m3fn)[:, 16:116], scale, wq, wscale, F32))
    wide[:, 17:117] = as8(q)
    assert torch.equal(want, linear_q8(wide.view(torch.float8_e4m3fn)[:, 17:117], scale, wq, wscale, F32))
    same = q[:1].expand(200, 100)
    assert torch.equal(linear_q8(same, scale[:1].expand(200), wq, wscale, F32), want[:1].expand(200, 120))
    pairs = torch.stack([scale, scale], 1)[:, 0]
    assert torch.equal(want, linear_q8(q, pairs, wq, wscale, F32))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [linear_q8(q, scale, wq, wscale, F32) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_infinite_and_nan_scales_stay_in_their_row():
    q, scale, wq, wscale = operands(130, 64, 40)
    want = linear_q8(q, scale, wq, wscale, F32)
    scale[3], scale[7] = float("nan"), float("inf")
    out = linear_q8(q, scale, wq, wscale, F32)
    keep = torch.ones(130, dtype=torch.bool, device=dev)
    keep[[3, 7]] = False
    assert torch.equal(out[keep], want[keep]) and torch.isnan(out[3]).all() and not torch.isfinite(out[7]).any()


def test_empty_rows():
    q, scale, wq, wscale = operands(4, 64, 40)
    assert linear_q8(q[:0], scale[:0], wq, wscale).shape == (0, 40)
    a, b = quantise(torch.empty(0, 24, device=dev))
    assert a.shape == (0, 24) and b.shape == (0,)


@pytest.mark.parametrize("rows", [16, 300])
def test_captured_and_replayed(rows):
    x = torch.randn(rows, 256, device=dev, dtype=BF16)
    wq, wscale = quantise(torch.randn(512, 256, device=dev))
    s = torch.cuda.Stream()
    run = lambda: linear_q8(*quantise(x), wq, wscale)  # noqa: E731
    with torch.cuda.stream(s):
        run()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = run()
    for seed in (1, 2):
        x.copy_(torch.randn(rows, 256, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert torch.equal(out, run())


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("n,d", [(1, 1), (5, 17), (300, 1152), (9, 5001), (2, 16384)])
def test_quantise(n, d, dt):
    """The rule bit for bit, and every value within half a code."""
    x = (torch.randn(n, d, device=dev) * torch.exp(torch.randn(n, 1, device=dev))).to(dt)
    q, scale = quantise(x)
    top = x.float().abs().amax(1, keepdim=True)
    want = (x.float() * (448.0 / top)).to(torch.float8_e4m3fn)
    assert torch.equal(q.contiguous().view(torch.uint8), want.view(torch.uint8))
    assert q.stride(0) % 16 == 0 or n == 1
    s64 = top.double()[:, 0] / 448
    assert ((scale.double() - s64).abs() <= s64 * 2 ** -23).all()
    off = (q.double() * s64[:, None] - x.double()).abs()
    assert (off <= x.double().abs() * (2 ** -4 + 2 ** -22) + s64[:, None] * 2 ** -9.99).all()
    zero, zscale = quantise(torch.zeros(3, 40, device=dev, dtype=dt))
    assert not zero.float().any() and torch.isfinite(zscale).all()
    bad = torch.ones(2, 40, device=dev, dtype=dt)
    bad[0, 3], bad[1, 4] = float("nan"), float("inf")
    assert not torch.isfinite(quantise(bad)[1]).any()


def test_refusals():
    q, scale, wq, wscale = operands(8, 64, 40)
    f = torch.zeros(8, 64, device=dev, requires_grad=True)
    for call in (lambda: linear_q8(q, scale, wq[:, :32], wscale), lambda: linear_q8(q, scale[:4], wq, wscale),
                 lambda: linear_q8(q, scale, wq, wscale.half()), lambda: linear_q8(q.float(), scale, wq, wscale),
                 lambda: linear_q8(q, scale, wq, wscale, torch.float64), lambda: linear_q8(q, scale, wq.cpu(), wscale),
                 lambda: linear_q8(q, scale.clone().requires_grad_(True), wq, wscale), lambda: quantise(f),
                 lambda: quantise(f.detach()[0]), lambda: linear_q8(q[:, :0], scale, wq[:, :0], wscale)):
        with pytest.raises(RuntimeError):
            call()
    torch.compile(lambda: linear_q8(q, scale, wq, wscale), fullgraph=True)()
    assert _ext.device_status() == 0
