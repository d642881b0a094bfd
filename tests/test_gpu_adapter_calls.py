"""Calls of the adapter and clipping operators that have to be refused, or to leave
what they do not own as it was, and what an error says."""
from __future__ import annotations

import pytest
import torch

import fp_emulation as fp
from fp_emulation import _lib
from test_gpu_adapters import _data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [20, 300, 40000])
def test_the_error_names_the_first_bad_row(rows, monkeypatch):
    """Wherever it stands: rows are counted by 32 warps, each in a stretch of its own."""
    from fp_emulation import ozaki

    for bad in (0, rows // 3, rows - 1):
        index = torch.zeros(rows, dtype=torch.int32, device="cuda")
        index[bad:] = 3
        monkeypatch.setattr(ozaki, "_CHECK_MODE", "off")
        for _ in range(5):
            fp.prepare_rows(index, 3)
            torch.cuda.synchronize()
            code, where, _, detail = _lib.device_error(clear=True)
            assert (code, where, detail) == (_lib.FPEMU_ERR_INVALID, _lib.WHERE_ADAPTER_INDEX, bad)


@pytest.mark.parametrize("rows", [20, 400])
def test_scales_changed_before_the_backward_pass(rows):
    x, A, B, base, dy, scale, index = _data(rows, 3, 16, 24, 4, torch.float64)
    x.requires_grad_(True)
    y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    scale.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x, dy)
    scale.mul_(0.5)
    again, = torch.autograd.grad(fp.adapter_matmul(x, A, B, index, base=base, scale=scale), x, dy)
    assert torch.equal(again, want)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    x, A, B, base, dy, scale, index = _data(20, 3, 16, 24, 4, torch.float64)
    with fwd.dual_level():
        operands = [x, A, B, base, scale]
        for i, t in enumerate(operands):
            dual = operands[:i] + [fwd.make_dual(t, torch.ones_like(t))] + operands[i + 1:]
            with pytest.raises(RuntimeError, match="forward-mode"):
                fp.adapter_matmul(*dual[:3], index, base=dual[3], scale=dual[4])
        with pytest.raises(RuntimeError, match="forward-mode"):
            fp.grad_norm([x, fwd.make_dual(dy, torch.ones_like(dy))])
        with pytest.raises(RuntimeError, match="forward-mode"):
            fp.clip_grads([fwd.make_dual(dy, torch.ones_like(dy))], 1.0)
        plain = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    assert torch.equal(plain, fp.adapter_matmul(x, A, B, index, base=base, scale=scale))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: fp.adapter_matmul(t, A, B, index), (x,), (x,))


def test_prepared_rows_of_another_shape():
    x, A, B, base, _, scale, index = _data(12, 3, 16, 24, 4, torch.float64)
    want = fp.adapter_matmul(x, A, B, index)
    square = fp.prepare_rows(index.view(4, 3), 3)
    with pytest.raises(RuntimeError, match="prepared for"):
        fp.adapter_matmul(x.view(3, 4, 16), A, B, square)
    with pytest.raises(RuntimeError, match="prepared for"):
        fp.adapter_matmul(x.view(3, 4, 16), A, B, fp.prepare_rows(index[:4], 3, (4, 3)))
    assert torch.equal(fp.adapter_matmul(x.view(4, 3, 16), A, B, square).view(12, 24), want)
    assert torch.equal(fp.adapter_matmul(x, A, B, square), want)  # rows in their order
    assert torch.equal(fp.adapter_matmul(x.view(2, 6, 16), A, B, fp.prepare_rows(index, 3)).view(12, 24), want)


def test_the_callers_gradient_stays_as_it_was():
    """create_graph: base's gradient is dy itself, which is not the operator's to change."""
    x, A, B, base, dy, scale, index = _data(12, 3, 16, 24, 4, torch.float64)
    for t in (x, A, B, base):
        t.requires_grad_(True)
    y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    dx, dbase = torch.autograd.grad(y, (x, base), dy, create_graph=True)
    assert not dy.requires_grad and torch.equal(dbase, dy)
    with pytest.raises(RuntimeError, match="once"):
        dx.sum().backward()
    weight = torch.ones_like(dy).requires_grad_(True)
    y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    dbase, = torch.autograd.grad((y * weight).sum(), base, create_graph=True)
    assert torch.equal(torch.autograd.grad(dbase.sum(), weight)[0], torch.ones_like(dy))  # linear in dy


def test_out_without_columns():
    x, A, B, base, _, scale, index = _data(12, 3, 16, 0, 4, torch.float64)
    out = torch.empty(12, 0, dtype=torch.float64, device="cuda")
    assert fp.adapter_matmul(x, A, B, index, base=base, out=out) is out
    layer = fp.add_adapters(fp.Linear(16, 0, device="cuda"), 3, rank=4)
    with torch.no_grad(), fp.use_adapters(layer, index):
        assert layer(x).shape == (12, 0)


@pytest.mark.parametrize("rows", [12, 300])
def test_out_over_the_ids_or_the_scales(rows):
    x, A, B, base, _, scale, index = _data(rows, 3, 16, 4, 4, torch.float64)
    out = torch.zeros(rows, 4, dtype=torch.float64, device="cuda")
    ids = out.view(torch.int64).flatten()[:rows]
    ids.copy_(index)
    if rows <= _lib.FPEMU_ADAPTER_FEW_ROWS:  # more are copied as they are grouped
        with pytest.raises(RuntimeError, match="overlaps"):
            fp.adapter_matmul(x, A, B, ids, out=out)
    want = fp.adapter_matmul(x, A, B, index)
    assert torch.equal(fp.adapter_matmul(x, A, B, fp.prepare_rows(ids, 3), out=out), want)
    with pytest.raises(RuntimeError, match="overlaps"):
        fp.adapter_matmul(x, A, B, index, scale=out.flatten()[4:7], out=out)
    leaf = torch.zeros_like(out).requires_grad_(True)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        fp.adapter_matmul(x, A, B, index, out=leaf)
    with torch.no_grad():
        assert torch.equal(fp.adapter_matmul(x, A, B, index, out=leaf), want)
