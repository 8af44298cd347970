"""The vocabulary cross entropy (B200) against the definition in float64 on the same inputs: loss and
gradients over types, sizes from one row up, odd rows and vocabularies, reductions, ignored rows, the
rows whose logits leave the target far behind, and its refusals.

Bounds, derived for the kernels' steps (U = one rounding of the operands' type, 2^-8 bf16, 2^-11 f16):
  logits  fp32 accumulation of K products in steps of 16: (K/16 + 8) 2^-23 sum_k |x_k w_k|
  loss    the largest logit error of the row, and a few fp32 roundings of the result
  dx      U of the result (its rounding), and U + that logit error + 2^-14 of the sum of its terms'
          magnitudes (the exponentials' rounding; fp32 sums over V, exponential and factors)
  dw      the same with 2 U (the exponentials' and the scaled rows' roundings)
  f16     e = 2^10 p has a smallest step of 2^-24, so p is off by up to 2^-35 where it is that small;
          the scaled rows by 2^-24 of the largest |g|; results by their own smallest step
"""
import ctypes

import pytest
import torch

import _ext
from gpu_util import capi
from linear_cross_entropy import KEEP_ROWS, linear_cross_entropy, reference

pytestmark = pytest.mark.gpu
dev = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inputs(N, V, K, dtype, seed=0, std=1.0, ignored=0.0, lift=0.3):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, K, generator=g) * K ** -0.5 * std).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    x = (torch.randn(N, K, generator=g) + lift * K ** 0.5 * torch.rand(N, 1, generator=g) * w[t].float()).to(dtype)
    t = torch.where(torch.rand(N, generator=g) < ignored, -100, t)
    return x.to(dev), w.to(dev), t.to(dev)


def exact(x, w, t, scale=1.0, z=0.0, up=None, ignore=-100):
    """(loss rows, dx, dw, and the bounds' magnitudes) in float64; up: the gradient of each row's loss."""
    X, W = x.double(), w.double()
    live = t != ignore
    tt = torch.where(live, t, 0).long()
    X = torch.where(live[:, None], X, 0.0)
    L = X @ W.t() * scale
    lse = torch.logsumexp(L, 1)
    rows = torch.arange(len(t), device=dev)
    loss = torch.where(live, lse - L[rows, tt] + z * lse * lse, 0.0)
    spread = (X.abs().float() @ W.abs().float().t()).amax(1).double() * abs(scale)
    lerr = (x.shape[1] / 16 + 8) * 2.0 ** -23 * spread
    out = {"loss": loss, "lerr": torch.where(live, lerr, 0.0)}
    if up is None:
        return out
    up = torch.where(live, up.double(), 0.0) * torch.ones_like(loss)
    soft = torch.exp(L - lse[:, None]) * ((1 + 2 * z * lse) * up)[:, None]
    # the magnitudes of the two parts of dl: the target's own term apart from the others
    mag = soft.abs()
    pt = torch.exp(L[rows, tt] - lse)
    mag[rows, tt] = ((1 - pt).abs() + (2 * z * lse * pt).abs()) * up.abs()
    dl = soft
    dl[rows, tt] -= up
    s = abs(scale)
    out.update(dx=dl @ W * scale, dw=dl.t() @ X * scale, mdx=mag @ W.abs() * s, mdw=mag.t() @ X.abs() * s,
               gtop=up.abs().max(), wsum=W.abs().sum(0) * s, psum=(mag.t() @ torch.ones_like(loss))[:, None] * s,
               xsum=X.abs().sum(0) * s, up=up)
    return out


def check_loss(got, e, rows=True):
    bound = 4 * e["lerr"] + 2.0 ** -20 * (1 + e["loss"].abs())
    if rows:
        err = (got.double() - e["loss"]).abs()
        assert torch.all(err <= bound), (err - bound).max()
    return bound


def check_grads(dx, dw, e, dtype, parts=("dx", "dw")):
    U, f16 = UNIT[dtype], dtype == torch.float16
    tiny = 2.0 ** -25 if f16 else 2.0 ** -133
    le = e["lerr"].max() * 4 + 2.0 ** -14
    if "dx" in parts:
        assert dx.dtype == dtype
        bound = 1.01 * U * e["dx"].abs() + (U + le) * e["mdx"] + tiny
        if f16:
            bound = bound + 2.0 ** -35 * e["up"].abs()[:, None] * e["wsum"] * 1.1
        err = (dx.double() - e["dx"]).abs()
        assert torch.all(err <= bound), ("dx", (err / bound).max())
    if "dw" in parts:
        assert dw.dtype == dtype
        bound = 1.01 * U * e["dw"].abs() + (2 * U + le) * e["mdw"] + tiny
        if f16:
            bound = bound + e["gtop"] * (2.0 ** -35 * 1.1 * e["xsum"] + 2.0 ** -24 * e["psum"] / e["gtop"].clamp(min=1e-30))
        err = (dw.double() - e["dw"]).abs()
        assert torch.all(err <= bound), ("dw", (err / bound).max())


def run(x, w, t, up=None, **kw):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, **kw)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    return loss.detach(), dx, dw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,K", [(1, 1, 8), (1, 1000, 64), (2, 257, 72), (17, 256, 512), (129, 1009, 320),
                                   (256, 4096, 1152), (257, 10007, 512), (300, 255, 264), (1500, 3001, 200),
                                   (2049, 1100, 1152), (5, 40000, 96)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_and_gradients(N, V, K, dtype, reduction):
    x, w, t = inputs(N, V, K, dtype, N + V + K, ignored=0.15 if N > 4 else 0.0)
    gen = torch.Generator().manual_seed(1)
    up = torch.rand(N, generator=gen).to(dev) if reduction == "none" else None
    kept = max(1, int((t != -100).sum()))
    weight = up if reduction == "none" else torch.tensor(1.0 / kept if reduction == "mean" else 1.0, device=dev)
    e = exact(x, w, t, up=weight)
    loss, dx, dw = run(x, w, t, up, reduction=reduction)
    bound = check_loss(loss, e, rows=reduction == "none")
    assert loss.dtype == torch.float32
    if reduction != "none":
        want = e["loss"].sum() / (kept if reduction == "mean" else 1)
        assert abs(loss.double() - want) <= bound.sum() / (kept if reduction == "mean" else 1)
    check_grads(dx, dw, e, dtype)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, t, reduction=reduction), loss)
    assert _ext.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [100, KEEP_ROWS + 60])
def test_scale_z_loss_and_upstream(N, dtype):
    V, K, scale, z = 2003, 256, 1 / 16, 1e-2
    x, w, t = inputs(N, V, K, dtype, 3, std=16.0, ignored=0.1)
    kept = int((t != -100).sum())
    e = exact(x, w, t, scale, z, torch.tensor(3.5 / kept, device=dev))
    loss, dx, dw = run(x, w, t, torch.tensor(3.5, device=dev), scale=scale, z_loss=z)
    assert abs(loss.double() - e["loss"].sum() / kept) <= (check_loss(loss, e, False).sum() + 2 * z * (e["lerr"] * 12).sum()) / kept
    check_grads(dx, dw, e, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction,N", [("none", 700), ("sum", KEEP_ROWS + 5)])
def test_rows_whose_target_is_far_below(dtype, reduction, N):
    """Logits of a spread of hundreds: the target's exponential underflows against the maximum (a loss of
    up to several hundred), in some 256-row blocks and not in others; losses stay finite and exact."""
    V, K = 1111, 64
    x, w, t = inputs(N, V, K, dtype, 5, lift=0.0)
    x = x.clone()
    x[3] *= 100
    x[130] *= 40
    x[600:620] *= 60
    up = torch.ones(N, device=dev)
    e = exact(x, w, t, up=up)
    assert e["loss"][3] > 60 and e["loss"][600:620].max() > 60
    loss, dx, dw = run(x, w, t, up if reduction == "none" else None, reduction=reduction)
    if reduction == "none":
        check_loss(loss, e)
    assert torch.isfinite(loss).all()
    check_grads(dx, dw, e, dtype)


def test_confident_rows_keep_their_small_loss():
    """Targets with a probability of 1 - 1e-6 and closer to 1: the loss is log1p of a small sum, not the
    difference of two large numbers, so it is right to a relative error, not only an absolute one."""
    # entry 7 alone has column 0, where row i holds 14 to 60; the other logits are 0
    N, V, K = 64, 500, 64
    w = torch.zeros(V, K)
    w[7, 0] = 1.0
    w[:, 1] = 0.5
    w[7, 1] = 0.0
    x = torch.zeros(N, K)
    x[:, 0] = torch.linspace(14, 60, N)
    x, w, t = x.bfloat16().to(dev), w.bfloat16().to(dev), torch.full((N,), 7, device=dev)
    small = torch.log1p((V - 1) * torch.exp(-x[:, 0].double()))
    loss, dx, dw = run(x, w, t, torch.ones(N, device=dev), reduction="none")
    # logits here are exact in fp32; the sum of 499 exponentials of 2 ulp each and a few roundings
    assert torch.all((loss.double() - small).abs() <= 2.0 ** -18 * small), ((loss.double() - small) / small).abs().max()
    # d loss / d x_0 = -(1 - p_t) here, however small: one rounding to bf16
    assert torch.all((dx[:, 0].double() - torch.expm1(-small)).abs() <= 2.0 ** -8 * 1.02 * small)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3.38e38])
@pytest.mark.parametrize("N", [60, KEEP_ROWS + 300])
def test_ignored_rows_may_hold_anything(bad, N):
    x, w, t = inputs(N, 700, 128, torch.bfloat16, 9)
    t[5::7] = -100
    e = exact(x, w, t, up=torch.ones(N, device=dev))
    dirty = x.clone()
    dirty[5::7] = bad
    loss, dx, dw = run(dirty, w, t, reduction="sum")
    assert abs(loss.double() - e["loss"].sum()) <= check_loss(loss, e, False).sum()
    check_grads(dx, dw, e, torch.bfloat16)
    assert not dx[5::7].any()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N", [40, KEEP_ROWS])
def test_no_row_left(N, reduction):
    x, w, t = inputs(N, 300, 64, torch.bfloat16, 2)
    t = torch.full_like(t, 7)
    loss, dx, dw = run(x, w, t, torch.ones(N, device=dev) if reduction == "none" else None, ignore_index=7,
                       reduction=reduction)
    assert not loss.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("N", [50, KEEP_ROWS])
def test_targets_outside_the_vocabulary_are_nan(N):
    x, w, t = inputs(N, 300, 64, torch.bfloat16, 2)
    for wrong in (300, -1, 2 ** 40):
        t2 = t.clone()
        t2[10] = wrong
        loss, dx, dw = run(x, w, t2, torch.ones(N, device=dev), reduction="none")
        assert loss[10].isnan() and torch.isfinite(loss[:10]).all() and torch.isfinite(loss[11:]).all()
        assert dx[10].isnan().all() and torch.isfinite(dx[:10]).all()
        assert run(x, w, t2)[0].isnan()


def test_several_chunks_of_rows():
    """A vocabulary of a million entries: chunks of 256 rows, fp32 sums of dw over them."""
    N, V, K = 600, 1_000_003, 64
    x, w, t = inputs(N, V, K, torch.bfloat16, 4, ignored=0.1)
    up = torch.rand(N, device=dev)
    e = exact(x, w, t, up=up)
    loss, dx, dw = run(x, w, t, up, reduction="none")
    check_loss(loss, e)
    check_grads(dx, dw, e, torch.bfloat16)


@pytest.mark.parametrize("N", [200, KEEP_ROWS + 1])
def test_one_gradient_only(N):
    x, w, t = inputs(N, 900, 136, torch.bfloat16, 6)
    loss, dx, dw = run(x, w, t)
    a = x.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, t), a)[0], dx)
    b = w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, b, t), b)[0], dw)


def test_strided_operands_and_int32_targets():
    N, V, K = 130, 260, 64
    x, w, t = inputs(N, V, K, torch.bfloat16, 7)
    wide = torch.randn(N, 2 * K + 1, device=dev, dtype=torch.bfloat16)
    wide[:, 1:K + 1] = x
    off = torch.zeros(V * K + 1, device=dev, dtype=torch.bfloat16)
    off[1:] = w.reshape(-1)
    t2 = torch.stack([t, t], 1).int()[:, 0]
    a, b = run(x, w, t), run(wide[:, 1:K + 1], off[1:].view(V, K), t2)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_same_bits_every_time_and_on_another_stream():
    x, w, t = inputs(1200, 5000, 256, torch.bfloat16, 8)
    a = run(x, w, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = run(x, w, t)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_the_two_backward_paths_agree():
    """Gradients formed in the forward and gradients from logits computed again: the same products."""
    N, V, K = KEEP_ROWS, 2000, 128
    x, w, t = inputs(N, V, K, torch.bfloat16, 11)
    e = exact(x, w, t, up=torch.full((N,), 2.0, device=dev))
    a = run(x, w, t, torch.tensor(2.0, device=dev), reduction="sum")
    b = run(x, w, t, torch.full((N,), 2.0, device=dev), reduction="none")
    for g in (a, b):
        check_grads(g[1], g[2], e, torch.bfloat16)


def test_gradient_against_differences():
    """Central differences of the fp32 sum of losses along random directions, in f16 values with a step of
    2^-4 (exact in f16 around the inputs' grid of 2^-8): the third derivative along a direction of unit
    entries is bounded by (sum |w|)^3 of the logits' spread; measured in float64 below instead of assumed."""
    N, V, K = 33, 200, 64
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(N, K, generator=g) * 256).round().div(256).half().to(dev)
    w = (torch.randn(V, K, generator=g) * 32).round().div(256).half().to(dev)
    t = torch.randint(0, V, (N,), generator=g).to(dev)
    _, dx, dw = run(x, w, t, reduction="sum")
    h = 2.0 ** -4

    def total(a, b):
        with torch.no_grad():
            return linear_cross_entropy(a, b, t, reduction="none").double().sum()

    def total64(a, b):
        return exact(a, b, t)["loss"].sum()

    for seed in range(3):
        d = torch.randint(0, 2, x.shape, generator=torch.Generator().manual_seed(seed)).to(dev).half() * 2 - 1
        quot = (total(x + h * d, w) - total(x - h * d, w)) / (2 * h)
        quot64 = (total64((x + h * d), w) - total64((x - h * d), w)) / (2 * h)
        e = exact(x, w, t, up=torch.ones(N, device=dev))
        truncation = (quot64 - (e["dx"] * d.double()).sum()).abs()
        noise = 33 * 2 * 2e-5 / (2 * h) + 2.0 ** -10 * e["mdx"].sum()
        assert abs((dx.double() * d.double()).sum() - quot) <= truncation + noise


def test_a_loss_changed_in_place_and_no_gradient_of_the_gradient():
    for N in (64, KEEP_ROWS):
        x, w, t = inputs(N, 300, 64, torch.bfloat16, 15)
        want = run(x, w, t, torch.tensor(0.25, device=dev))
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(a, b, t)
        loss /= 4
        assert torch.allclose(loss, want[0] / 4)
        for g, h in zip(torch.autograd.grad(loss, (a, b)), want[1:]):
            assert torch.equal(g, h)
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(linear_cross_entropy(a, b, t), a, create_graph=True)


def test_compiled_matches_eager():
    for N in (100, KEEP_ROWS):
        x, w, t = inputs(N, 600, 64, torch.bfloat16, 12)
        a, b = x.requires_grad_(True), w.requires_grad_(True)
        for reduction in ("mean", "none"):
            fn = torch.compile(lambda a, b: linear_cross_entropy(a, b, t, z_loss=1e-3, reduction=reduction), fullgraph=True)
            p, q = linear_cross_entropy(a, b, t, z_loss=1e-3, reduction=reduction), fn(a, b)
            assert torch.equal(p, q)
            up = torch.ones_like(p)
            for g, h in zip(torch.autograd.grad(p, (a, b), up), torch.autograd.grad(q, (a, b), up)):
                assert torch.equal(g, h)


def test_in_a_cuda_graph():
    x, w, t = inputs(300, 1000, 128, torch.bfloat16, 13)
    up = torch.ones(300, device=dev)
    want = run(x, w, t, up, reduction="none")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(x, w, t, up, reduction="none")
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x, w, t, up, reduction="none")
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    del graph


def test_matches_the_torch_expression():
    x, w, t = inputs(500, 800, 128, torch.bfloat16, 14, ignored=0.2)
    for reduction in ("mean", "sum", "none"):
        a = linear_cross_entropy(x, w, t, 0.7, z_loss=1e-3, reduction=reduction)
        assert torch.allclose(a, reference(x, w, t, 0.7, z_loss=1e-3, reduction=reduction), rtol=1e-4, atol=1e-4)


def test_empty():
    for reduction in ("mean", "sum", "none"):
        x = torch.empty(0, 64, device=dev, dtype=torch.bfloat16)
        w = torch.randn(50, 64, device=dev).bfloat16()
        t = torch.empty(0, dtype=torch.long, device=dev)
        loss, dx, dw = run(x, w, t, torch.empty(0, device=dev) if reduction == "none" else None, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and not loss.any()
        assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def test_refusals():
    x, w, t = inputs(10, 20, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(RuntimeError, match="2-D"):
        linear_cross_entropy(x[0], w, t)
    with pytest.raises(RuntimeError, match="w must be"):
        linear_cross_entropy(x, w[:, :32], t)
    with pytest.raises(RuntimeError, match="one dtype"):
        linear_cross_entropy(x, w.half(), t)
    with pytest.raises(RuntimeError, match="unsupported"):
        linear_cross_entropy(x.float(), w.float(), t)
    with pytest.raises(RuntimeError, match="unsupported"):
        linear_cross_entropy(x[:, :60].contiguous(), w[:, :60].contiguous(), t)
    with pytest.raises(RuntimeError, match="targets must be"):
        linear_cross_entropy(x, w, t[:5])
    with pytest.raises(RuntimeError, match="int32 or int64"):
        linear_cross_entropy(x, w, t.float())
    with pytest.raises((RuntimeError, NotImplementedError)):
        linear_cross_entropy(x.cpu(), w, t)
    # the C ABI: a workspace that is too small or missing is refused before anything is launched
    vp, i64, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
    loss = torch.empty(10, device=dev)
    call = lambda ws, size: capi().krsi_linear_ce_fwd(  # noqa: E731
        vp(x.data_ptr()), vp(w.data_ptr()), vp(t.data_ptr()), 64, vp(loss.data_ptr()), vp(0), vp(0), vp(0), vp(0), vp(0), vp(ws),
        ctypes.c_size_t(size), i64(10), i64(20), i64(64), f32(1.0), i64(-100), f32(0.0), 0, 1, vp(0))
    assert call(0, 1 << 20) == 4 and call(t.data_ptr(), 16) == 4
