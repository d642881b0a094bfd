"""adapter_matmul at the ends of what it takes: nothing to sum or to write, shared
and expanded operands, ragged columns of padded rows, the length where few rows
become many, thousands of adapters, offsets past 32 bits, several threads, captured
training, and the Linear layers' block.  Tolerances are those of
test_gpu_adapters."""
from __future__ import annotations

import threading

import pytest
import torch

import fp_emulation as fp
from test_gpu_adapters import DTYPES, _close, _data, _formula, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_no_inputs_or_no_outputs(dtype, rows):
    for k, m in ((0, 9), (9, 0), (0, 0)):
        x, A, B, base, dy, scale, index = _data(rows, 3, k, m, 4, dtype)
        for t in (x, A, B, base):
            t.requires_grad_(True)
        y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        assert torch.equal(y, base) and torch.equal(fp.adapter_matmul(x.detach(), A.detach(), B.detach(), index, scale=scale),
                                                    torch.zeros_like(base))
        dx, dA, dB, dbase = torch.autograd.grad(y, (x, A, B, base), dy)
        assert torch.equal(dbase, dy)
        for g, t in ((dx, x), (dA, A), (dB, B)):
            assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("rows", [40, 500])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_shared_and_expanded_operands(dtype, rows):
    """One pair of factors for every adapter, one row of x for every request, base a bias."""
    n, k, m, r = 3, 64, 72, 8
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, dtype)
    x1, A1, B1, bias = (t[:1].detach().clone().requires_grad_(True) for t in (x, A, B, base))
    wide = [x1.expand(rows, k), A1.expand(n, r, k), B1.expand(n, m, r), bias.expand(rows, m)]
    y = fp.adapter_matmul(*wide[:3], index, base=wide[3], scale=scale)
    full = [t.detach().contiguous().requires_grad_(True) for t in wide]
    y2 = fp.adapter_matmul(*full[:3], index, base=full[3], scale=scale)
    assert torch.equal(y, y2)
    _close(y.detach(), *_formula(*[t.detach() for t in full], scale, index)[:2], k + r, dtype)
    got = torch.autograd.grad(y, wide, dy)
    want = torch.autograd.grad(y2, full, dy)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    shared = torch.autograd.grad(fp.adapter_matmul(*[t.expand(w.shape) for t, w in zip((x1, A1, B1), wide)], index,
                                                   base=bias.expand(rows, m), scale=scale), (x1, A1, B1, bias), dy)
    for s, w in zip(shared, want):
        assert torch.equal(s, w.sum(0, keepdim=True))


@pytest.mark.parametrize("r", [3, 16, 40, 72])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_ragged_columns_of_padded_rows(dtype, r):
    """Rows that start aligned and end within 16 bytes, NaN behind their ends."""
    for rows in (7, 270):
        for k, m in ((33, 17), (200, 131), (1, 257)):
            x, A, B, base, _, scale, index = _data(rows, 3, k, m, r, dtype, seed=r + k)
            padded = []
            for t in (x, A, B, base):
                wide = torch.full(t.shape[:-1] + ((t.shape[-1] + 31) // 16 * 16,), float("nan"), dtype=dtype, device="cuda")
                wide[..., :t.shape[-1]] = t
                padded.append(wide[..., :t.shape[-1]])
            out = torch.full((rows, m + 15), 7.0, dtype=dtype, device="cuda")
            y = fp.adapter_matmul(*padded[:3], index, base=padded[3], scale=scale, out=out[:, :m])
            _close(y, *_formula(x, A, B, base, scale, index)[:2], k + r, dtype)
            assert (out[:, m:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_where_few_rows_become_many(dtype):
    x, A, B, base, _, scale, index = _data(260, 5, 96, 160, 16, dtype)
    for rows in (1, 255, 256, 257, 260):
        want, mag = _formula(x[:rows], A, B, base[:rows], scale, index[:rows])[:2]
        for ids in (index[:rows], index[:rows].long(), fp.prepare_rows(index[:rows], 5)):
            _close(fp.adapter_matmul(x[:rows], A, B, ids, base=base[:rows], scale=scale), want, mag, 112, dtype)


@pytest.mark.parametrize("rows", [256, 3000])
def test_the_most_adapters(rows):
    n, k, m, r = 65000, 8, 12, 2
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, torch.float64)
    index[0], index[1], index[2] = n - 1, n - 1, 0
    i = index.long().clamp(min=0)
    on = (index >= 0).double()[:, None]
    for t in (x, A, B):
        t.requires_grad_(True)
    y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    plain = base + on * scale[i][:, None] * torch.einsum("tnr,trk,tk->tn", B[i], A[i], x)
    # 10 products, each below 10 in magnitude, in either order
    assert (y - plain).abs().max() < 2.0 ** -53 * 10 * 20 * 50
    for g, w in zip(torch.autograd.grad(y, (x, A, B), dy), torch.autograd.grad(plain, (x, A, B), dy)):
        assert (g - w).abs().max() < 2.0 ** -53 * 10 * 20 * 50


def test_offsets_past_32_bits():
    rows, k = 70000, 32768  # 2.3e9 elements
    index = torch.arange(rows, device="cuda", dtype=torch.int32) // 64 % 3 - 1
    last = slice(rows - 200, rows)
    for wide_x in (True, False):
        kk, m, r = (k, 8, 4) if wide_x else (8, k, 4)
        _, A, B, _, _, scale, _ = _data(1, 2, kk, m, r, torch.bfloat16)
        x = torch.zeros((rows, kk), dtype=torch.bfloat16, device="cuda")
        x[last] = torch.randn((200, kk), device="cuda").to(torch.bfloat16)
        base = torch.ones((rows, m), dtype=torch.bfloat16, device="cuda")
        dy = torch.zeros_like(base)
        dy[last] = 1
        want, mag, u, ua = _formula(x[last], A, B, base[last], scale, index[last])
        for t in (x, A, B):
            t.requires_grad_(True)
        y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        _close(y.detach()[last], want, mag, kk + r, torch.bfloat16)
        assert (y.detach()[:rows - 200] == 1).all()
        dx, dA, dB = torch.autograd.grad(y, (x, A, B), dy)
        with torch.no_grad():
            dxw, dxm, v, va = _formula(dy[last], B.transpose(1, 2), A.transpose(1, 2), None, scale, index[last])
            _close(dx[last], dxw, dxm, m + r, torch.bfloat16)
            assert not dx[:rows - 200].any()
            for i in range(2):
                t = index[last] == i
                _close(dA[i], v[t].T @ x[last][t].double(), va[t].T @ x[last][t].double().abs(), m + 200, torch.bfloat16)
                _close(dB[i], dy[last][t].double().T @ u[t], dy[last][t].double().abs().T @ ua[t], kk + 200, torch.bfloat16)
        del x, y, dx, base, dy


def test_threads_at_once():
    """First calls of several threads, each on its own stream."""
    sets = [_data(rows, 4, 128, 200, r, dtype, seed=rows) for rows, r, dtype in
            ((90, 100, torch.float64), (500, 100, torch.float32), (30, 20, torch.float16), (2000, 60, torch.bfloat16))]
    torch.cuda.synchronize()
    got, errors = [None] * len(sets), []

    def work(i):
        try:
            x, A, B, base, _, scale, index = sets[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [fp.adapter_matmul(x, A, B, index, base=base, scale=scale) for _ in range(5)]
                torch.cuda.current_stream().synchronize()
        except Exception as exc:  # noqa: BLE001
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for ys, (x, A, B, base, _, scale, index) in zip(got, sets):
        want = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        assert all(torch.equal(y, want) for y in ys)


@pytest.mark.parametrize("rows", [32, 600])
def test_captured_training(rows):
    """Forward, gradients and clipping in one graph, replayed on new data."""
    n, k, m, r = 4, 96, 128, 12
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, torch.float32, "mixed", 1)
    A.requires_grad_(True), B.requires_grad_(True)

    def step():
        y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        return fp.clip_grads(torch.autograd.grad(y, (A, B), dy), 0.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads, norm = step()
    for seed in (2, 3):
        new = _data(rows, n, k, m, r, torch.float32, "mixed", seed)
        for t, s in ((x, new[0]), (dy, new[4]), (index, new[6])):
            t.copy_(s)
        graph.replay()
        want, want_norm = step()
        assert torch.equal(norm, want_norm) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_block_of_linear_layers():
    """The ids are read as the block begins; blocks nest; inference mode and capture within."""
    model = fp.add_adapters(_model(5), 3, rank=2)
    for layer in model:
        if isinstance(layer, fp.Linear):
            torch.nn.init.normal_(layer.adapters.B)
    x = torch.randn(30, 2, device="cuda", dtype=torch.float64)
    a, b = (torch.full((30,), i, device="cuda") for i in (0, 2))

    def run(ids):
        with fp.use_adapters(model, ids), torch.no_grad():
            return model(x)

    want_a, want_b = run(a), run(b)
    assert not torch.equal(want_a, want_b)
    ids = a.clone()
    with fp.use_adapters(model, ids), torch.inference_mode():
        ids.copy_(b)
        assert torch.equal(model(x), want_a)
        with fp.use_adapters(model, b):
            assert torch.equal(model(x), want_b)
        assert torch.equal(model(x), want_a)
    with pytest.raises(TypeError):
        with fp.use_adapters(model, [0] * 30):
            pass
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(ids)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(ids)
    for source, want in ((a, want_a), (b, want_b)):
        ids.copy_(source)
        graph.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("adapters", [1, 3])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_long_batches_of_narrow_layers(dtype, adapters):
    """Few columns and many rows: the gradients' sums come in several parts."""
    rows, k, m, r = 30011, 40, 24, 5
    x, A, B, base, dy, scale, index = _data(rows, adapters, k, m, r, dtype, "mixed", 8)
    index[-7000:] = adapters - 1
    for t in (x, A, B):
        t.requires_grad_(True)

    def grads(*wanted):
        y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        return torch.autograd.grad(y, wanted, dy)

    dx, dA, dB = grads(x, A, B)
    assert all(torch.equal(a, b) for a, b in zip(grads(x, A, B), (dx, dA, dB)))
    only_A, = grads(A)
    only_B, = grads(B)
    with torch.no_grad():
        _, _, u, ua = _formula(x, A, B, base, scale, index)
        dxw, dxm, v, va = _formula(dy, B.transpose(1, 2), A.transpose(1, 2), None, scale, index)
        _close(dx, dxw, dxm, m + r, dtype)
        for i in range(adapters):
            t = index == i
            for got in (dA[i], only_A[i]):
                _close(got, v[t].T @ x[t].double(), va[t].T @ x[t].double().abs(), m + rows, dtype)
            for got in (dB[i], only_B[i]):
                _close(got, dy[t].double().T @ u[t], dy[t].double().abs().T @ ua[t], k + rows, dtype)
