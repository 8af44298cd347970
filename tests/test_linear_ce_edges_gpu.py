"""The vocabulary cross entropy (B200) at the limits of its types and paths, against float64."""
import ctypes

import pytest
import torch

import _ext
from gpu_util import capi
from linear_cross_entropy import KEEP_ROWS, linear_cross_entropy
from test_linear_ce_gpu import UNIT, check_grads, check_loss, exact, inputs, run

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("N,reduction", [(40, "mean"), (300, "none"), (KEEP_ROWS + 60, "mean"), (KEEP_ROWS + 60, "none")])
def test_f16_rows_scaled_far_up_by_the_z_loss(N, reduction):
    """x up to 1e4 and log-sum-exps in the hundreds with z = 0.1: x (1 + 2 z lse) is far above f16's 65504, the
    gradients are not.  Row 5 is four times smaller, so that the factors differ from row to row."""
    V, K, z, scale, dtype = 700, 64, 0.1, 0.1, torch.float16
    x, w, t = inputs(N, V, K, dtype, 21, ignored=0.1, lift=0.0)
    x = (x.float() * 1000).clamp(-1e4, 1e4).half()
    x[5] *= 0.25
    t[5] = 3
    kept = int((t != -100).sum())
    up = torch.rand(N, device=dev) / kept if reduction == "none" else None
    e = exact(x, w, t, scale, z, up if up is not None else torch.tensor(1.0 / kept, device=dev))
    loss, dx, dw = run(x, w, t, up, scale=scale, z_loss=z, reduction=reduction)
    live = t != -100
    L = torch.where(live[:, None], x.double(), 0.0) @ w.double().t() * scale
    lse = torch.logsumexp(L, 1)
    p = torch.exp(L - lse[:, None]) * live[:, None]
    soft = (e["up"] * (1 + 2 * z * lse)).abs()
    assert (x.double().abs().amax(1) * (1 + 2 * z * lse)).max() > 2 * 65504
    # the row's own |p - 1| 2 z lse term: the loss moves by 1 + 2 z lse for an error of lse
    tol = (4 * e["lerr"] + 2.0 ** -20 * (1 + lse)) * (1 + 2 * z * lse) + 2.0 ** -20 * e["loss"].abs()
    if reduction == "none":
        assert torch.all((loss.double() - e["loss"]).abs() <= tol)
    else:
        assert abs(loss.double() - e["loss"].sum() / kept) <= tol.sum() / kept
    # as in test_linear_ce_gpu: the result's rounding; the exponentials' and the scaled rows' (dw) and the logits'
    # errors on the magnitudes; e's smallest step (p off by 2^-35) and the scaled rows' (2^-24 of the largest factor)
    U, le = UNIT[dtype], e["lerr"].max() * 4 + 2.0 ** -14
    bdx = 1.01 * U * e["dx"].abs() + (U + le) * e["mdx"] + 2.0 ** -25 + 1.1 * 2.0 ** -35 * soft[:, None] * e["wsum"]
    bdw = (1.01 * U * e["dw"].abs() + (2 * U + le) * e["mdw"] + 2.0 ** -25
           + soft.max() * (1.1 * 2.0 ** -35 * e["xsum"] + 2.0 ** -24 * scale * p.sum(0)[:, None]))
    assert torch.isfinite(dw).all() and torch.isfinite(dx).all()
    assert torch.all((dx.double() - e["dx"]).abs() <= bdx)
    assert torch.all((dw.double() - e["dw"]).abs() <= bdw)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("N", [64, KEEP_ROWS])
def test_logits_far_from_zero_lose_nothing(N):
    """Two entries whose logits are 1024 and 1024 + k / 64, both exact in fp32: the loss log1p(exp(k / 64)) is right
    to what its exponential and logarithm cost, with no rounding of a logit's own size (2^-14 in log2 units here:
    4e-5 of the exponential) in between."""
    x, w = torch.zeros(N, 64), torch.zeros(2, 64)
    k = (torch.arange(N) * 37 % 509 - 254).float()
    x[:, 0], w[:, 0] = 64.0, 16.0
    x[:, 1], w[1, 1] = k / 64, 1.0
    t = torch.zeros(N, dtype=torch.long)
    x, w, t = x.bfloat16().to(dev), w.bfloat16().to(dev), t.to(dev)
    want = torch.log1p(torch.exp(x[:, 1].double()))
    with torch.no_grad():
        loss = linear_cross_entropy(x, w, t, reduction="none")
    # l - ref: one rounding at up to 4 log2(e) = 5.8; 2 units each of the exponentials, factors and logarithm
    assert torch.all((loss.double() - want).abs() <= 2.0 ** -19 * want), ((loss.double() - want).abs() / want).max()


@pytest.mark.parametrize("N", [60, KEEP_ROWS])
@pytest.mark.parametrize("scale", [0.0, -0.5])
def test_scales_of_zero_and_below(N, scale):
    """A scale of 0 (every logit 0: the loss is log V) and a negative one, with a ragged vocabulary."""
    x, w, t = inputs(N, 333, 64, torch.bfloat16, 8, ignored=0.1)
    e = exact(x, w, t, scale, up=torch.ones(N, device=dev))
    loss, dx, dw = run(x, w, t, torch.ones(N, device=dev), scale=scale, reduction="none")
    check_loss(loss, e)
    check_grads(dx, dw, e, torch.bfloat16)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("N,V", [(1100, 300_001), (8192, 500), (8193, 500), (8300, 40_000)])
def test_the_loss_has_the_same_bits_with_and_without_gradients(N, V, reduction):
    """Rows on both sides of the reductions' border, and chunks with gradients where there are none without."""
    x, w, t = inputs(N, V, 64, torch.bfloat16, 17, ignored=0.1)
    loss = run(x, w, t, reduction=reduction)[0]
    with torch.no_grad():
        rows = linear_cross_entropy(x, w, t, reduction="none")
        assert torch.equal(linear_cross_entropy(x, w, t, reduction=reduction), loss)
    count = int((t != -100).sum()) if reduction == "mean" else 1
    # rows added in float64, one rounding
    assert abs(loss.double() - rows.double().sum() / count) <= 2.0 ** -23 * loss.double()


def workspace(N, V, K, mode):
    size = ctypes.c_size_t(0)
    rc = capi().krsi_linear_ce_workspace_size(ctypes.c_int64(N), ctypes.c_int64(V), ctypes.c_int64(K), mode, ctypes.byref(size))
    assert rc == 0
    return size.value


def test_the_losses_workspace_is_bounded():
    """The loss alone holds a chunk's partial sums (256 MB at most, or 256 rows') and under 32 bytes a row."""
    for N, V in ((1, 100), (4096, 131072), (32768, 131072), (1 << 20, 131072), (1 << 24, 32768), (1 << 20, 1 << 26)):
        part = max(1 << 28, 256 * 16 * ((V + 255) // 256))
        assert workspace(N, V, 64, 0) <= part + 32 * N + 4096


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("N", [600, KEEP_ROWS + 276])
def test_losses_of_several_chunks(N, bits):
    """A vocabulary of 8.4 million entries cuts the rows of the loss alone into chunks of 256."""
    V, K = 8_400_003, 8
    g = torch.Generator(device=dev).manual_seed(2)
    w = torch.randn(V, K, generator=g, device=dev).bfloat16()
    x = torch.randn(N, K, generator=g, device=dev).bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[3::11] = -100
    with torch.no_grad():
        rows = linear_cross_entropy(x, w, t if bits == 64 else t.int(), reduction="none")
        total = linear_cross_entropy(x, w, t if bits == 64 else t.int(), reduction="sum")
    W = w.double()
    want = torch.zeros(N, dtype=torch.float64, device=dev)
    for i in range(0, N, 64):
        L = x[i:i + 64].double() @ W.t()
        want[i:i + 64] = torch.logsumexp(L, 1) - L.gather(1, t[i:i + 64].clamp(min=0)[:, None])[:, 0]
        del L
    want = torch.where(t != -100, want, 0.0)
    # sums of exponentials: 128 of a half tile, 2 V / 256 / 32 half tiles a lane, 8 more; the logits' own 2^-20
    bound = (128 + V // 4096 + 8) * 2.0 ** -24 + 2.0 ** -20 * (1 + want)
    assert torch.all((rows.double() - want).abs() <= bound), (rows.double() - want).abs().max()
    assert torch.equal(total, rows.double().sum().float())
    assert _ext.device_status() == 0


@pytest.mark.parametrize("N", [1, 600])
def test_one_gradient_takes_its_own_workspace_alone(N):
    """The weight's fp32 rows and sorted targets are held for dw only, dx's shares for dx only; and each gradient alone
    has the bits that it has beside the other, on every path."""
    V, K = 20_000, 512
    both, no_dw, no_dx = (workspace(N, V, K, 2 + f) for f in (0, 8, 4))
    assert no_dw < both - 4 * min(N, V) * K + 4096 and no_dx <= both
    chunk = 256 * ((N + 255) // 256)      # e and x' of a chunk, and at most one share of dx per 8 blocks of 64 entries
    assert no_dw <= 64 * N + chunk * (2 * (V + 64) + 2 * K) + 4 * chunk * K * (V // 512 + 1) + 8192
    assert workspace(N, V, K, 1 + 8) <= workspace(N, V, K, 1) and workspace(N, V, K, 1 + 4) <= workspace(N, V, K, 1)
    x, w, t = inputs(N, V, K, torch.bfloat16, 3)
    up = torch.rand(N, device=dev)
    loss, dx, dw = run(x, w, t, up, reduction="none")
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, t, reduction="none"), a, up)[0], dx)
    assert torch.cuda.max_memory_allocated() - held <= no_dw + 4 * N * K + (1 << 21)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, b, t, reduction="none"), b, up)[0], dw)


def test_the_weights_sums_go_by_the_rows_where_those_are_fewer():
    """One row over a large vocabulary used to hold fp32 sums for every entry of w (604 MB here)."""
    assert workspace(1, 131072, 1152, 2) < 256 * 131072 * 2 + (16 << 20)   # the exponentials of 256 rows, and little else
    assert workspace(3000, 1000, 512, 2) < workspace(3000, 3001, 512, 2)


@pytest.mark.parametrize("N,V", [(40, 5000), (512, 5000), (513, 5000), (700, 701), (700, 700), (700, 699), (500, 33),
                                 (40, 70_001), (512, 70_001), (513, 70_001), (2000, 70_001)])
def test_tokens_that_occur_often(N, V):
    """A few tokens that hold most of the rows (runs over many chunks of the sorted sum) among single ones, with more
    tokens than rows and fewer; the sums' rows are those of the tokens that occur."""
    x, w, t = inputs(N, V, 136, torch.bfloat16, 31)
    often = torch.randint(0, 3, (N,), generator=torch.Generator().manual_seed(4)).to(dev) * (V // 3 + 1) % V
    t = torch.where(torch.arange(N, device=dev) % 4 == 0, t, often)
    t[1::13] = -100
    up = torch.rand(N, device=dev)
    e = exact(x, w, t, up=up)
    loss, dx, dw = run(x, w, t, up, reduction="none")
    check_loss(loss, e)
    check_grads(dx, dw, e, torch.bfloat16)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction,z", [("mean", 0.0), ("sum", 1e-3), ("none", 0.0)])
def test_gradients_over_several_chunks(reduction, z, dtype):
    """A vocabulary that cuts 1100 rows into chunks of 768: gradients formed in the forward (mean, sum) and later
    (none), ignored rows in both chunks, and rows of both whose target lies far below another logit."""
    N, V, K = 1100, 300_001, 64
    x, w, t = inputs(N, V, K, dtype, 6, ignored=0.1, lift=0.0)
    x = x.clone()
    for r in (5, 700, 768, 900, N - 1):
        x[r] *= 40
        t[r] = r
    kept = int((t != -100).sum())
    up = torch.rand(N, device=dev) if reduction == "none" else None
    weight = up if reduction == "none" else torch.tensor(1.0 / kept if reduction == "mean" else 1.0, device=dev)
    e = exact(x, w, t, 1.0, z, weight)
    assert e["loss"][[5, 900]].max() > 60
    loss, dx, dw = run(x, w, t, up, z_loss=z, reduction=reduction)
    if reduction == "none":
        check_loss(loss, e)
    else:
        want = e["loss"].sum() / (kept if reduction == "mean" else 1)
        # (z: an error of lse counts 1 + 2 z lse times; lse is below 150 here)
        assert abs(loss.double() - want) <= 1.3 * check_loss(loss, e, False).sum() / (kept if reduction == "mean" else 1)
    check_grads(dx, dw, e, dtype)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [1272, 1280, 1288, 2048, 4104])
@pytest.mark.parametrize("N,reduction", [(70, "none"), (530, "mean"), (KEEP_ROWS + 3, "mean")])
def test_wide_rows(N, reduction, K, dtype):
    """Rows around and past the 1280 columns that a warp has under way at once, on all three gradient paths."""
    V = 601
    x, w, t = inputs(N, V, K, dtype, K, ignored=0.1)
    kept = int((t != -100).sum())
    up = torch.rand(N, device=dev) if reduction == "none" else None
    e = exact(x, w, t, up=up if up is not None else torch.tensor(1.0 / kept, device=dev))
    loss, dx, dw = run(x, w, t, up, reduction=reduction)
    if reduction == "none":
        check_loss(loss, e)
    else:
        assert abs(loss.double() - e["loss"].sum() / kept) <= check_loss(loss, e, False).sum() / kept
    check_grads(dx, dw, e, dtype)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_more_rows_than_the_joins_block_reduces(reduction):
    N, V, K = 8300, 300, 64
    x, w, t = inputs(N, V, K, torch.bfloat16, 12, ignored=0.2)
    kept = int((t != -100).sum())
    up = torch.rand(N, device=dev) if reduction == "none" else None
    weight = up if reduction == "none" else torch.tensor(1.0 / kept if reduction == "mean" else 1.0, device=dev)
    e = exact(x, w, t, up=weight)
    loss, dx, dw = run(x, w, t, up, reduction=reduction)
    bound = check_loss(loss, e, rows=reduction == "none")
    if reduction != "none":
        k = kept if reduction == "mean" else 1
        assert abs(loss.double() - e["loss"].sum() / k) <= bound.sum() / k
    check_grads(dx, dw, e, torch.bfloat16)


@pytest.mark.parametrize("N", [511, 512, 513])
def test_both_sides_of_the_one_launch_sum(N):
    x, w, t = inputs(N, 1500, 72, torch.bfloat16, N, ignored=0.1)
    up = torch.rand(N, device=dev)
    e = exact(x, w, t, up=up)
    loss, dx, dw = run(x, w, t, up, reduction="none")
    check_loss(loss, e)
    check_grads(dx, dw, e, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_in_several_chunks(dtype):
    """Up to 512 rows, so that the targets' sums need no sort, over a vocabulary that leaves 256 to a chunk."""
    N, V, K = 300, 1_000_003, 64
    x, w, t = inputs(N, V, K, dtype, 14, ignored=0.1)
    t[7::20] = t[0]
    up = torch.rand(N, device=dev)
    e = exact(x, w, t, up=up)
    loss, dx, dw = run(x, w, t, up, reduction="none")
    check_loss(loss, e)
    check_grads(dx, dw, e, dtype)
