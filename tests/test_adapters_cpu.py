"""Adapters and gradient clipping without a GPU: what the entry points refuse,
how ids are spread over rows, and the plan's layout."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import fp_emulation as fp
from fp_emulation import _lib
from fp_emulation.adapters import _check_out, _spread_index
from fp_emulation.gradients import _dense, _norm_code


def _lists(n):
    return (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)(), (ctypes.c_int32 * n)()


def test_python_refusals_without_a_gpu():
    x, A, B = torch.zeros(3, 4, dtype=torch.float64), torch.zeros(2, 1, 4, dtype=torch.float64), torch.zeros(2, 5, 1, dtype=torch.float64)
    with pytest.raises(TypeError):
        fp.adapter_matmul(x.to(torch.int32), A, B, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        fp.adapter_matmul(x, A, B, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError):
        fp.prepare_rows(torch.zeros(3, dtype=torch.float32), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp.prepare_rows(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(ValueError):
        fp.prepare_rows(torch.zeros(3, dtype=torch.int32), 0)
    with pytest.raises(ValueError):
        fp.Adapters(2, 4, 5, rank=0)
    with pytest.raises(ValueError):
        fp.Adapters(2, 4, 5, rank=129)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp.grad_norm([x])
    with pytest.raises(ValueError):
        fp.grad_norm([x], norm_type=3.0)
    with pytest.raises(ValueError):
        fp.clip_grads([x], -1.0)
    with pytest.raises(ValueError):
        fp.clip_grads([x], float("nan"))
    with pytest.raises(TypeError):
        fp.grad_norm([x.to(torch.int64)])
    with pytest.raises(TypeError):
        fp.grad_norm([3.0])
    with pytest.raises(RuntimeError, match="no Linear with adapters"):
        with fp.use_adapters(torch.nn.Sequential(torch.nn.Linear(2, 2)), torch.zeros(1, dtype=torch.int32)):
            pass


def test_empty_lists_have_norm_zero():
    assert fp.grad_norm([]) == 0
    assert fp.clip_grads([], 1.0)[0] == []
    p = torch.nn.Parameter(torch.ones(3))
    assert fp.clip_grad_norm_([p], 1.0) == 0
    assert [_norm_code(p) for p in (1, 2, 2.0, math.inf)] == [1, 2, 2, 0]


def test_ids_spread_over_rows():
    ids = torch.tensor([3, -1])
    assert _spread_index(ids, torch.Size([2])).tolist() == [3, -1]
    assert _spread_index(ids, torch.Size([2, 3])).tolist() == [[3] * 3, [-1] * 3]
    with pytest.raises(RuntimeError):
        _spread_index(ids, torch.Size([3, 2]))
    with pytest.raises(RuntimeError):
        _spread_index(ids.view(1, 2), torch.Size([2]))


def test_out_must_not_meet_an_input():
    buf = torch.zeros(100)
    x, out = buf[:20].view(4, 5), buf[20:40].view(4, 5)
    assert _check_out(out, out.shape, x, None, (x,)).data_ptr() == out.data_ptr()
    assert _check_out(out, out.shape, x, out, (x,)) is not None
    with pytest.raises(RuntimeError, match="overlaps an input"):
        _check_out(buf[19:39].view(4, 5), out.shape, x, None, (x,))
    with pytest.raises(RuntimeError, match="base"):
        _check_out(out, out.shape, x, buf[21:41].view(4, 5), (x,))
    with pytest.raises(RuntimeError, match="rows"):
        _check_out(buf[40:45].expand(4, 5), out.shape, x, None, (x,))
    with pytest.raises(RuntimeError, match="shape"):
        _check_out(out, torch.Size([5, 4]), x, None, (x,))


def test_dense_means_each_element_once():
    t = torch.zeros(4, 6, 5)
    assert _dense(t) and _dense(t.permute(2, 0, 1)) and _dense(t[:1]) and _dense(torch.zeros(())) and _dense(t[1:3])
    assert not _dense(t[:, ::2]) and not _dense(t[..., :3]) and not _dense(torch.zeros(1).expand(4))


def test_plan_size_and_c_refusals():
    lib = _lib.load()
    # start words (n + 3 rounded to 4), slots twice (4 words each, rows // 64 + n + 2), 4 words, rows
    for rows, n in ((0, 1), (1, 1), (63, 5), (64, 5), (1000, 64), (1 << 20, 65000)):
        assert lib.fpemu_adapter_plan_size(rows, n) == 4 * ((n + 3 + 3) // 4 * 4 + 8 * (rows // 64 + n + 2) + 4 + rows)
    assert lib.fpemu_adapter_plan_size(-1, 1) == 0 and lib.fpemu_adapter_plan_size(1, 0) == 0
    assert lib.fpemu_adapter_plan(None, 4, 1, 1, None, 0, None) == _lib.FPEMU_ERR_WORKSPACE
    assert lib.fpemu_adapter_plan(None, 2, 1, 1, None, 0, None) == _lib.FPEMU_ERR_INVALID

    def matmul(dtype=0, rows=4, k=8, n=8, rank=2, adapters=2, x=16, y=16, x_row=8, y_row=8, index=16, nbytes=4, plan=None):
        return lib.fpemu_adapter_matmul(dtype, rows, k, n, rank, adapters, x, x_row, 16, 16, 8, 16, 16, 2, None, 0,
                                        y, y_row, None, 1.0, index, nbytes, plan, None, None, 0, None)

    bad, unsupported = _lib.FPEMU_ERR_INVALID, _lib.FPEMU_ERR_UNSUPPORTED
    assert matmul(dtype=4) == bad and matmul(rows=-1) == bad and matmul(x=None) == bad and matmul(y=None) == bad
    assert matmul(x_row=-1) == bad and matmul(y_row=7) == bad
    assert matmul(index=None) == bad and matmul(nbytes=2) == bad and matmul(rows=257) == bad
    assert matmul(rank=0) == unsupported and matmul(rank=129) == unsupported and matmul(adapters=0) == unsupported
    assert matmul(rows=0) == 0

    def backward(rows=4, plan=16, v=16, dx=16, x=16, stride=8):
        return lib.fpemu_adapter_backward(0, rows, 8, 8, 2, 2, x, stride, 16, 16, 8, 16, 16, 2, 16, 8, None, 1.0, plan, 16, v,
                                          dx, 16, 16, None, 0, None)

    assert backward(plan=None) == bad and backward(v=None) == bad and backward(v=8) == bad
    assert backward(x=None) == bad and backward(stride=-1) == bad


def test_clip_c_refusals():
    lib = _lib.load()
    bad = _lib.FPEMU_ERR_INVALID

    def clip(ranges, outs=None, dtype=1, norm_type=2, max_norm=1.0, norm=64):
        src, dst, numel, dt = _lists(len(ranges))
        for i, (a, n) in enumerate(ranges):
            src[i], numel[i], dt[i] = a, n, dtype
            dst[i] = a if outs is None else outs[i]
        return lib.fpemu_clip_grads(len(ranges), src, dst, numel, dt, norm_type, max_norm, norm, 0, None, 0, None)

    assert clip([(4096, 10)], dtype=4) == bad
    assert clip([(4096, -1)]) == bad and clip([(None, 3)]) == bad
    assert clip([(4096, 10)], norm_type=3) == bad and clip([(4096, 10)], max_norm=-1.0) == bad
    assert clip([(4096, 10)], max_norm=math.nan) == bad and clip([(4096, 10)], norm=None) == bad
    # the same tensor twice; one that starts inside another; an output over another's input
    assert clip([(4096, 10), (4096, 10)]) == bad and b"overlaps" in lib.fpemu_last_error()
    assert clip([(4096, 10), (4132, 4)]) == bad
    assert clip([(4096, 10), (8192, 10)], [8192, 16384]) == bad
    assert clip([(4096, 10), (8192, 10)], [4100, 16384]) == bad
    # disjoint lists pass the check (and end at the missing device or workspace)
    assert clip([(4096, 10), (4136, 10)]) != bad
    assert clip([(4096, 10), (4096, 10)], [8192, 16384]) != bad
