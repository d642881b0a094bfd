"""One use_adapters block on several streams, from several threads and beside graph
captures: every use sees the block's ids, ordered after the copy of them."""
from __future__ import annotations

import threading

import pytest
import torch

import fp_emulation as fp
from test_gpu_adapters import _data, _model

pytestmark = pytest.mark.gpu

ROWS = 700  # more than the kernel groups by itself: the plan is used


def _adapted(seed):
    model = fp.add_adapters(_model(seed), 5, rank=3)
    for layer in model:
        if isinstance(layer, fp.Linear):
            torch.nn.init.normal_(layer.adapters.B)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(ROWS, 2, generator=gen, device="cuda", dtype=torch.float64)
    ids = torch.randint(-1, 5, (ROWS,), generator=gen, device="cuda")
    return model, x, ids


def _step(model, x):
    """A result and the gradients of every parameter."""
    y = model(x)
    return (y.detach(), *torch.autograd.grad(y.sum(), list(model.parameters())))


def _same(a, b):
    return all(torch.equal(s, t) for s, t in zip(a, b))


def test_one_block_from_threads_with_a_stream_each():
    model, x, ids = _adapted(1)
    with fp.use_adapters(model, ids):
        want, frozen = _step(model, x), model(x).detach()
    torch.cuda.synchronize()
    errors, got = [], {}
    late = torch.full_like(ids, -1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda._sleep(50_000_000)  # the copies of the ids below wait behind this
    late.copy_(ids)
    with fp.use_adapters(model, late):
        def work(i):
            try:
                with torch.cuda.stream(streams[i]):
                    with torch.no_grad():
                        first = model(x)
                    got[i] = [first] + [_step(model, x) for _ in range(5)]
                    torch.cuda.current_stream().synchronize()
            except Exception as exc:  # noqa: BLE001
                errors.append(exc)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not errors
    for first, *steps in got.values():
        assert torch.equal(first, frozen) and all(_same(s, want) for s in steps)


def _warm(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()


def test_capture_inside_a_block_then_eager_then_replays():
    model, x, ids = _adapted(2)
    with fp.use_adapters(model, ids), torch.no_grad():
        want = model(x)
        _warm(lambda: model(x))
    graph = torch.cuda.CUDAGraph()
    source = ids.clone()
    with fp.use_adapters(model, source), torch.no_grad():
        with torch.cuda.graph(graph):  # the first use of this shape in the block
            y = model(x)
        assert torch.equal(model(x), want)  # before any replay: its own plan
        graph.replay()
        assert torch.equal(y, want)
        assert torch.equal(model(x), want)
    source.fill_(-1)
    del source
    for _ in range(3):  # memory that the block let go of is used again
        torch.full((ROWS,), 4, dtype=torch.int64, device="cuda"), torch.full((4 * ROWS,), 3, device="cuda")
    y.zero_()
    graph.replay()
    assert torch.equal(y, want)  # a graph keeps the ids of its block


def test_two_captures_in_one_block():
    model, x, ids = _adapted(3)
    with fp.use_adapters(model, ids):
        want = _step(model, x)
        _warm(lambda: _step(model, x))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with fp.use_adapters(model, ids):
        results = []
        for graph in graphs:
            with torch.cuda.graph(graph):
                results.append(_step(model, x))
        graphs[1].replay()  # the first graph has not run
        assert _same(results[1], want)
        graphs[0].replay()
        assert _same(results[0], want)


def test_what_a_capture_made_is_refused_outside():
    model, x, ids = _adapted(4)
    A = B = None
    x2, A, B, base, _, scale, index = _data(ROWS, 4, 16, 24, 3, torch.float64)
    with fp.use_adapters(model, ids), torch.no_grad():
        want = model(x)
        _warm(lambda: model(x))
    _warm(lambda: fp.adapter_matmul(x2, A, B, fp.prepare_rows(index, 4), base=base, scale=scale))
    graph = torch.cuda.CUDAGraph()
    block = fp.use_adapters(model, ids)
    A.requires_grad_(True)
    with torch.cuda.graph(graph):
        rows = fp.prepare_rows(index, 4)
        y = fp.adapter_matmul(x2, A, B, rows, base=base, scale=scale)
        block.__enter__()
        with torch.no_grad():
            model(x)
    with pytest.raises(RuntimeError, match="capture"):
        fp.adapter_matmul(x2, A.detach(), B, rows, base=base, scale=scale)
    with pytest.raises(RuntimeError, match="capture"):
        torch.autograd.grad(y.sum(), A)
    with pytest.raises(RuntimeError, match="capture"):
        model(x)
    block.__exit__(None, None, None)
    with fp.use_adapters(model, ids), torch.no_grad():
        assert torch.equal(model(x), want)
