"""C entry points of the adapter and clipping operators refuse addresses that are not
multiples of their element sizes: the kernels' loads would fault.  No GPU needed: the
checks come before the device is asked for (and where there is one, the calls that pass
them end at the missing workspace)."""
from __future__ import annotations

import ctypes

import pytest

from fp_emulation import _lib

SIZES = {0: 8, 1: 4, 2: 2, 3: 2}


@pytest.mark.parametrize("dtype", SIZES)
def test_adapter_pointers(dtype):
    lib = _lib.load()
    e = SIZES[dtype]
    good = dict(x=64, A=64, B=64, base=64, y=64, scales=64, index=64, plan=64, u=64)

    def matmul(**change):
        p = {**good, **change}
        return lib.fpemu_adapter_matmul(dtype, 4, 8, 8, 2, 2, p["x"], 8, p["A"], 16, 8, p["B"], 16, 2, p["base"], 8, p["y"], 8,
                                        p["scales"], 1.0, p["index"], 4, p["plan"], p["u"], None, 0, None)

    bad = _lib.FPEMU_ERR_INVALID
    assert matmul() in (_lib.FPEMU_ERR_NO_DEVICE, _lib.FPEMU_ERR_CUDA, _lib.FPEMU_ERR_WORKSPACE)  # no workspace is given
    for name in ("x", "A", "B", "base", "y"):
        assert matmul(**{name: 64 + e // 2}) == bad and b"aligned" in lib.fpemu_last_error()
    assert matmul(scales=68) == bad and matmul(index=66, plan=None) == bad and matmul(plan=72) == bad
    assert matmul(u=66 if e < 8 else 68) == bad

    good = dict(x=64, A=64, B=64, dy=64, scales=64, plan=64, dx=64, dA=64, dB=64)

    def backward(**change):
        p = {**good, **change}
        return lib.fpemu_adapter_backward(dtype, 4, 8, 8, 2, 2, p["x"], 8, p["A"], 16, 8, p["B"], 16, 2, p["dy"], 8,
                                          p["scales"], 1.0, p["plan"], 64, 64, p["dx"], p["dA"], p["dB"], None, 0, None)

    assert backward() != bad
    for name in ("x", "A", "B", "dy", "dx", "dA", "dB"):
        assert backward(**{name: 64 + e // 2}) == bad and b"aligned" in lib.fpemu_last_error()
    assert backward(scales=68) == bad and backward(plan=72) == bad
    assert lib.fpemu_adapter_plan(66, 4, 4, 2, 64, 1 << 20, None) == bad
    assert lib.fpemu_adapter_plan(68, 8, 4, 2, 64, 1 << 20, None) == bad


@pytest.mark.parametrize("dtype", SIZES)
def test_clipping_pointers(dtype):
    lib = _lib.load()
    e = SIZES[dtype]

    def clip(src=4096, dst=8192, norm=64, wide=1, numel=10):
        s, d = (ctypes.c_void_p * 1)(src), (ctypes.c_void_p * 1)(dst)
        n, t = (ctypes.c_int64 * 1)(numel), (ctypes.c_int32 * 1)(dtype)
        return lib.fpemu_clip_grads(1, s, d, n, t, 2, 1.0, norm, wide, None, 0, None)

    bad = _lib.FPEMU_ERR_INVALID
    assert clip() != bad and clip(norm=68, wide=0) != bad and clip(src=4097, numel=0) != bad
    assert clip(src=4096 + e // 2) == bad and clip(dst=8192 + e // 2) == bad
    assert clip(norm=68) == bad and clip(norm=66, wide=0) == bad
