"""Which plan a use_adapters block hands to which stream and capture, without a GPU:
streams, captures and plans are stand-ins that record what was asked of them."""
from __future__ import annotations

import contextlib
import math
import threading

import pytest
import torch

from fp_emulation import adapters


class Ids:
    """An index on a GPU."""

    def __init__(self):
        self.streams = []

    def clone(self):
        return self

    def get_device(self):
        return 0

    def record_stream(self, stream):
        self.streams.append(stream)


class Gpu:
    stream, capture = 1, 0

    def __init__(self, monkeypatch):
        self.made, self.waits, self.recorded = [], [], []
        gpu = self

        class Event:
            def record(self, stream):
                gpu.recorded.append(stream.handle)

        class Stream:
            def __init__(self):
                self.handle = gpu.stream

            def wait_event(self, event):
                gpu.waits.append(self.handle)

        def plan(index, n, lead):
            gpu.made.append((tuple(lead), n, gpu.stream, gpu.capture))
            return object()

        monkeypatch.setattr(adapters, "_raw_stream", lambda d: self.stream)
        monkeypatch.setattr(adapters, "_capture_id", lambda d: self.capture)
        monkeypatch.setattr(adapters, "PreparedRows", plan)
        monkeypatch.setattr(torch.cuda, "Event", Event)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream())


def _block(model=None):
    return adapters._ActiveRows(Ids(), model or torch.nn.Linear(1, 1))


def test_a_plan_for_each_stream_that_waits_for_the_ids(monkeypatch):
    gpu = Gpu(monkeypatch)
    active = _block()
    first = active.prepare((4, 3), 5)
    assert active.prepare((4, 3), 5) is first and len(gpu.made) == 1 and gpu.waits == []
    assert active.prepare((12,), 5) is not first and active.prepare((4, 3), 6) is not first
    gpu.stream = 2
    second = active.prepare((4, 3), 5)
    assert second is not first and gpu.waits == [2] and len(active.index.streams) == 1
    assert active.prepare((4, 3), 5) is second and gpu.waits == [2]
    gpu.stream = 1
    assert active.prepare((4, 3), 5) is first


def test_a_capture_keeps_its_plans_to_itself(monkeypatch):
    gpu = Gpu(monkeypatch)
    model = torch.nn.Linear(1, 1)
    active = _block(model)
    gpu.capture = 7
    captured = active.prepare((4,), 5)
    assert gpu.waits == [] and adapters._captured_ids[model] == [active.index]  # read by later replays
    gpu.capture = 8
    assert active.prepare((4,), 5) is not captured
    gpu.capture = 0
    assert active.prepare((4,), 5) is not captured
    gpu.capture = 7
    assert active.prepare((4,), 5) is captured


def test_a_block_begun_in_a_capture_is_refused_outside(monkeypatch):
    gpu = Gpu(monkeypatch)
    gpu.capture = 3
    active = _block()
    plan = active.prepare((4,), 5)
    gpu.stream = 2  # a stream that joined the capture
    assert active.prepare((4,), 5) is not plan and gpu.waits == [2]
    for other in (0, 4):
        gpu.capture = other
        with pytest.raises(RuntimeError, match="capture"):
            active.prepare((4,), 5)


def test_rows_prepared_in_a_capture_are_refused_outside(monkeypatch):
    now = [0]
    monkeypatch.setattr(adapters, "_capture_id", lambda d: now[0])
    rows = adapters.PreparedRows.__new__(adapters.PreparedRows)
    rows.index = Ids()
    for made, used, fine in ((0, 0, True), (0, 5, True), (5, 5, True), (5, 0, False), (5, 6, False)):
        rows.capture, now[0] = made, used
        with contextlib.nullcontext() if fine else pytest.raises(RuntimeError, match="capture"):
            rows.check_capture()


def test_threads_on_one_stream_share_one_plan(monkeypatch):
    gpu = Gpu(monkeypatch)
    active = _block()
    got, start = [], threading.Barrier(8)

    def work():
        start.wait()
        got.append(active.prepare((4,), 5))

    threads = [threading.Thread(target=work) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(gpu.made) == 1 and all(g is got[0] for g in got)


def test_forward_mode_tangents_are_seen():
    import torch.autograd.forward_ad as fwd

    t = torch.ones(3)
    adapters._no_tangents("call", t, None, 2.0)
    with fwd.dual_level():
        adapters._no_tangents("call", t, None, 2.0)
        with pytest.raises(RuntimeError, match="call has no forward-mode"):
            adapters._no_tangents("call", t, fwd.make_dual(t, t))


def test_out_without_rows_or_columns():
    for shape in ((3, 0), (0, 3), (2, 0, 3), (2, 3, 0)):
        out = torch.empty(shape)
        assert adapters._check_out(out, out.shape, out, None, ()).shape == (math.prod(shape[:-1]), shape[-1])


def test_a_model_is_copied_inside_a_block():
    import copy
    import pickle

    import fp_emulation as fp

    model = fp.add_adapters(torch.nn.Sequential(fp.Linear(2, 3)), 4, rank=1)
    ids = torch.tensor([1, -1, 3])
    with fp.use_adapters(model, ids):
        for twin in (copy.deepcopy(model), pickle.loads(pickle.dumps(model))):
            assert torch.equal(twin[0].active_rows.index, ids) and twin[0].active_rows is not model[0].active_rows
            assert torch.equal(twin[0].adapters.A, model[0].adapters.A)
    assert model[0].active_rows is None


def test_clipping_has_the_signature_it_names():
    import inspect

    import fp_emulation as fp

    ours, theirs = (inspect.signature(f).parameters for f in (fp.clip_grad_norm_, torch.nn.utils.clip_grad_norm_))
    assert list(ours) == list(theirs) and all(ours[n].default == p.default for n, p in theirs.items())
    p = torch.nn.Parameter(torch.ones(3))
    for foreach in (None, True, False):
        assert fp.clip_grad_norm_([p], 1.0, foreach=foreach) == 0
