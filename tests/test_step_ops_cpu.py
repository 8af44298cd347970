"""Host-side contract of the residual norm, the 8-bit projection and AdamW: signatures, fake (meta)
implementations, refusals without a device and the C ABI's argument checks, which return before any device work.
CPU only."""
import ctypes
import inspect

import pytest
import torch

from conftest import PKG

vp, i64, f32, f64, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_size_t
F32, BF16, F16 = 0, 1, 2
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(str(PKG / "lib" / "libkrsi_b200.so"))


def test_public_signatures():
    import adamw
    import add_rmsnorm
    import linear_q8

    names = lambda f: list(inspect.signature(f).parameters)  # noqa: E731
    assert names(add_rmsnorm.add_rmsnorm) == names(add_rmsnorm.add_rmsnorm_q8) == ["x2d", "res", "w", "eps"]
    assert names(linear_q8.linear_q8) == ["q", "scale", "wq", "wscale", "dtype"]
    assert names(linear_q8.quantise) == ["x2d"]
    assert names(adamw.adamw_step)[:5] == ["params", "grads", "exp_avgs", "exp_avg_sqs", "step"]
    for mod in (add_rmsnorm, linear_q8, adamw):
        assert callable(mod.reference) and callable(mod.selftest)


def test_fake_impls_give_the_shapes():
    import adamw  # noqa: F401

    ops = torch.ops.krsi
    m = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    x, w = m(6, 40), m(40)
    y, z, rstd = ops.add_rmsnorm_fwd(x, m(6, 40), w, 1e-6)
    assert y.shape == z.shape == (6, 40) and rstd.shape == (6,) and rstd.dtype == torch.float32
    assert ops.add_rmsnorm_fwd(x, None, w, 1e-6)[1].shape == (0, 40)
    dz, dw = ops.add_rmsnorm_bwd(y, None, z, w, rstd)
    assert dz.shape == (6, 40) and dw.shape == (40,)
    q, scale, z = ops.add_rmsnorm_q8(x, None, w, 1e-6)
    assert q.shape == (6, 40) and q.stride() == (48, 1) and q.dtype == E4M3 and scale.shape == (6,) and z.shape == (0, 40)
    wq, wscale = ops.quantise_rows(m(24, 40))
    out = ops.linear_q8(q, scale, wq, wscale, torch.float16)
    assert out.shape == (6, 24) and out.dtype == torch.float16


def test_lists_have_their_way_past_the_dispatcher():
    import adamw

    assert adamw.direct is not None and callable(adamw.direct.adamw_step)
    x, step = torch.zeros(4), torch.zeros((), dtype=torch.int64)
    args = ([x], [x], [x], [x], [], [], step, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0)
    assert adamw.direct.adamw_step(*args) is NotImplemented       # no CUDA tensors: the operator's to refuse
    with pytest.raises(TypeError):
        adamw.direct.adamw_step(x)


def test_cpu_tensors_are_rejected():
    import adamw
    import add_rmsnorm
    import linear_q8

    x, w, one = torch.zeros(4, 8), torch.ones(8), torch.ones(4)
    q = torch.zeros(4, 8).to(E4M3)
    step = torch.zeros((), dtype=torch.int64)
    for call in (lambda: add_rmsnorm.add_rmsnorm(x, x, w, 1e-6), lambda: add_rmsnorm.add_rmsnorm_q8(x, None, w, 1e-6),
                 lambda: linear_q8.quantise(x), lambda: linear_q8.linear_q8(q, one, q, one),
                 lambda: adamw.adamw_step([x], [x.clone()], [x.clone()], [x.clone()], step, lr=1e-3)):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()


def test_norm_argument_checks(lib):
    fwd, q8, rows = lib.krsi_add_rmsnorm_fwd, lib.krsi_add_rmsnorm_q8_fwd, lib.krsi_quantise_rows
    a = vp(16)

    def f(x=a, res=a, w=a, z=a, y=a, stat=a, n=4, d=8, xt=F32, wt=F32):
        return fwd(x, res, w, z, y, stat, i64(n), i64(d), f32(1e-6), xt, wt, vp(0))

    def g(x=a, res=a, w=a, z=a, q=a, stride=1 << 20, stat=a, n=4, d=8, xt=F32, wt=F32):
        return q8(x, res, w, z, q, i64(stride), stat, i64(n), i64(d), f32(1e-6), xt, wt, vp(0))

    for call in (f, g):
        assert call(n=0) == 0
        assert call(x=vp(0)) == call(w=vp(0)) == call(z=vp(0)) == call(stat=vp(0)) == call(n=-1) == call(d=0) == 1
        assert call(xt=7) == call(wt=5) == 1
        assert call(xt=BF16, wt=F16) == call(xt=F32, wt=BF16) == 2    # no such pair of types
        assert call(d=16388) == call(d=16385) == 2                    # wider than a row may be
    assert g(q=vp(0)) == g(stride=7) == 1
    assert rows(a, a, i64(16), a, i64(0), i64(8), F32, vp(0)) == 0
    assert rows(a, vp(0), i64(16), a, i64(4), i64(8), F32, vp(0)) == 1
    assert rows(a, a, i64(4), a, i64(4), i64(8), F32, vp(0)) == 1
    assert rows(a, a, i64(1 << 20), a, i64(4), i64(1 << 20), F32, vp(0)) == 2


def test_linear_q8_argument_checks(lib):
    def f(q=16, qs=64, s=16, wq=16, ws=64, wsc=16, out=16, rows=4, K=64, M=8, dt=BF16):
        return lib.krsi_linear_q8(vp(q), i64(qs), vp(s), vp(wq), i64(ws), vp(wsc), vp(out), i64(rows), i64(K), i64(M),
                                  dt, vp(0))

    assert f(rows=0, q=0) == 0
    assert f(q=0) == f(s=0) == f(wq=0) == f(wsc=0) == f(out=0) == f(rows=-1) == f(K=0) == f(M=0) == f(dt=9) == 1
    assert f(qs=48) == f(ws=32) == 1              # rows that overlap
    assert f(q=8) == f(wq=24) == f(qs=72) == f(ws=72) == 3
    assert f(rows=2 ** 31 - 1) == f(M=2 ** 31 - 1) == 2


class Tensor(ctypes.Structure):
    _fields_ = [(k, vp) for k in ("p", "g", "m", "v", "master", "exponents")] + \
        [("n", i64)] + [(k, ctypes.c_int) for k in ("p_dtype", "g_dtype", "state_bits", "reserved")]


def test_adamw_argument_checks(lib):
    need = size()
    assert lib.krsi_adamw_workspace_size(i64(3), ctypes.byref(need)) == 0 and need.value > 0
    assert lib.krsi_adamw_workspace_size(i64(-1), ctypes.byref(need)) == 1

    def f(tensor=None, count=1, step=16, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=0.0, norm=0, ws=16, room=1 << 20,
          **fields):
        t = Tensor(**{**dict(p=16, g=16, m=16, v=16, n=4, p_dtype=F32, g_dtype=F32, state_bits=32), **fields})
        return lib.krsi_adamw_step(ctypes.byref(t), i64(count), vp(step), vp(0), f64(1e-3), f64(beta1), f64(beta2),
                                   f64(eps), f64(0.0), f64(max_norm), vp(norm), vp(ws), size(room), vp(0))

    assert f(p=None) == f(g=None) == f(m=None) == f(v=None) == f(n=-1) == f(count=-1) == f(step=0) == 1
    assert f(p_dtype=5) == f(state_bits=16) == f(p_dtype=BF16, g_dtype=F16) == f(p_dtype=F32, g_dtype=BF16) == 1
    assert f(state_bits=8) == 1                                   # no exponents
    assert f(master=16) == 1                                      # of an fp32 parameter
    assert f(beta1=1.0) == f(beta2=-0.1) == f(eps=-1.0) == f(max_norm=-1.0) == f(max_norm=1.0) == f(max_norm=1e-60, norm=16) == 1
    assert f(state_bits=8, exponents=17) == 3 and f(ws=8) == 3
    assert f(ws=0) == f(room=64) == 4
