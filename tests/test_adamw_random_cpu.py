"""Host-side contract of AdamW's random rounding: the C ABI's flag, the operator's argument and the Python one.  CPU
only."""
import ctypes
import inspect

import pytest
import torch

from conftest import PKG

vp, i64, f64, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t


class Tensor(ctypes.Structure):
    _fields_ = [(k, vp) for k in ("p", "g", "m", "v", "master", "exponents")] + \
        [("n", i64)] + [(k, ctypes.c_int) for k in ("p_dtype", "g_dtype", "state_bits", "reserved")]


def test_c_abi_flag():
    lib = ctypes.CDLL(str(PKG / "lib" / "libkrsi_b200.so"))

    def f(state_bits, exponents=16, ws=16, reserved=0):
        t = Tensor(p=16, g=16, m=16, v=16, n=4, exponents=exponents, state_bits=state_bits, reserved=reserved)
        return lib.krsi_adamw_step(ctypes.byref(t), i64(1), vp(16), vp(0), f64(1e-3), f64(0.9), f64(0.999), f64(1e-8),
                                   f64(0.0), f64(0.0), vp(0), vp(ws), size(1 << 20), vp(0))

    # (a missing workspace is refused after the tensors have been looked at)
    assert f(8, ws=0) == f(8 + 256, ws=0) == f(32, ws=0) == f(8 + 256, ws=0, reserved=-1) == 4
    assert f(32 + 256, ws=0) == f(256, ws=0) == f(8 + 512, ws=0) == 1
    assert f(8 + 256, exponents=0) == 1 and f(8 + 256, exponents=17) == 3


def test_python_arguments():
    import adamw

    assert inspect.signature(adamw.adamw_step).parameters["rounding"].default is None
    x, step = torch.zeros(4), torch.zeros((), dtype=torch.int64)
    args = ([x], [x], [x], [x], [], [], step, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0)
    assert adamw.direct.adamw_step(*args, True) is NotImplemented and adamw.direct.adamw_step(*args) is NotImplemented
    with pytest.raises(TypeError):
        adamw.direct.adamw_step(*args, True, True)
    with pytest.raises(ValueError, match="rounding"):
        adamw.adamw_step([x], [x], [x], [x], step, lr=1e-3, rounding="up")
    schema = torch.ops.krsi.adamw_step.default._schema
    assert schema.arguments[-1].name == "random_m" and schema.arguments[-1].default_value is False
    meta = lambda t: t.to("meta")  # noqa: E731
    assert torch.ops.krsi.adamw_step(*[[meta(x)]] * 4, [], [], meta(step), *args[7:], True).shape == (0,)
