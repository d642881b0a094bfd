"""Low-rank adapters of many requests beside a shared projection.

A batch shares one projection ``base = x @ W.T`` (an emulated product, see
``fp_emulation.ozaki``); every row adds the low-rank product of its own adapter:

    y[t] = base[t] + scale_i * B[i] @ (A[i] @ x[t]),   i = index[t]

``adapter_matmul`` is the operator, with its gradients; ``prepare_rows`` groups
the rows of a batch by adapter once for all layers; ``Adapters`` holds the
factors as parameters, and ``add_adapters`` / ``use_adapters`` put them beside
the ``Linear`` layers of a model.  CUDA tensors only.  Nothing here has a
counterpart in the reference.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import threading
import weakref

import torch
from torch import nn
from torch.autograd import forward_ad

from fp_emulation import _lib
from fp_emulation.ozaki import _after_call, _dtype_bits, _on, _raw_stream, _require_cuda, _stream

_DTYPE_CODE = {torch.float64: _lib.FPEMU_DT_F64, torch.float32: _lib.FPEMU_DT_F32,
               torch.float16: _lib.FPEMU_DT_F16, torch.bfloat16: _lib.FPEMU_DT_BF16}


def _capture_id(device_index):
    """The graph capture that the current stream of a device belongs to, or 0."""
    number = ctypes.c_uint64(0)
    with _on(device_index):
        _lib.check(_lib.load().fpemu_capture_id(_raw_stream(device_index), ctypes.byref(number)), "capture")
    return number.value


class PreparedRows:
    """The rows of a batch grouped by adapter (``prepare_rows``): a snapshot of
    the index on the GPU, shared by every layer and by the backward pass."""

    def __init__(self, index, adapters, shape=None):
        if not isinstance(index, torch.Tensor) or index.dtype not in (torch.int32, torch.int64):
            raise TypeError("adapter ids are an int32 or int64 tensor")
        adapters = int(adapters)
        if not 1 <= adapters <= _lib.FPEMU_ADAPTER_MAX_COUNT:
            raise ValueError(f"{adapters} adapters; between 1 and {_lib.FPEMU_ADAPTER_MAX_COUNT} are supported")
        dev = _require_cuda(index)
        self.shape = index.shape if shape is None else torch.Size(shape)
        self.adapters = adapters
        self.index = _spread_index(index, self.shape).reshape(-1).clone()
        rows = self.index.numel()
        if rows > _lib.FPEMU_ADAPTER_MAX_ROWS:
            raise ValueError(f"{rows} rows; at most {_lib.FPEMU_ADAPTER_MAX_ROWS} are supported")
        lib = _lib.load()
        self.plan = torch.empty((lib.fpemu_adapter_plan_size(rows, adapters) // 4,), dtype=torch.int32, device=dev)
        with torch.cuda.device(dev):
            st = lib.fpemu_adapter_plan(self.index.data_ptr(), self.index.element_size(), rows, adapters,
                                        self.plan.data_ptr(), self.plan.numel() * 4, _stream(dev))
        _lib.check(st, "prepare_rows")
        _after_call("prepare_rows", dev)
        self.capture = _capture_id(dev.index)

    def check_capture(self):
        """A plan made in a capture is memory that nothing has written before the graph's first replay."""
        if self.capture and self.capture != _capture_id(self.index.get_device()):
            raise RuntimeError("rows prepared in the capture of a CUDA graph serve that capture alone")


def prepare_rows(index, adapters, shape=None):
    """Group the rows of a batch by adapter, once for every layer that the batch
    passes.  ``index`` (int32 or int64, on the GPU) holds each row's adapter,
    0 .. adapters - 1, or -1 for none; ``shape`` gives it the leading shape of the
    layers' inputs where it has fewer dimensions (one id for each request of a
    [requests, length, features] batch).  Later changes of ``index`` do not
    change the result.  On another stream than the one it was made on, wait for that
    one first, and keep the result until its uses have finished.  Made while a CUDA
    graph is captured, it serves that capture alone.  An id that is no adapter makes its
    rows NaN and raises ``FpemuError`` in the first call that ends after the kernel has
    seen it."""
    return PreparedRows(index, adapters, shape)


def _spread_index(index, shape):
    if index.shape == shape:
        return index
    if index.dim() > len(shape) or index.shape != shape[:index.dim()]:
        raise RuntimeError(f"adapter ids of shape {tuple(index.shape)} do not match rows of shape {tuple(shape)}")
    return index.reshape(index.shape + (1,) * (len(shape) - index.dim())).expand(shape)


def _no_tangents(what, *tensors):
    """Refuses forward-mode differentiation, which the kernels would drop in silence."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative")


def _last_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _packed_like(t, shape):
    """A new packed tensor of t's type (the cheapest way there is to make one)."""
    return torch.empty_like(t) if t.shape == shape and t.is_contiguous() else t.new_empty(shape)


def _launch(x, A, B, base, y, scale, rows, index, u):
    """One fpemu_adapter_matmul on the current stream of x's device (2-D x, base and y)."""
    dev = x.device
    d = dev.index
    lib = _lib.load()
    code, count = _DTYPE_CODE[x.dtype], x.shape[0]
    adapters, rank, k = A.shape
    plan = work = None  # few rows are grouped inside the kernel; more go by the plan
    size = 0
    with _on(d):
        if count > _lib.FPEMU_ADAPTER_FEW_ROWS:
            plan = rows.plan.data_ptr()
            size = lib.fpemu_adapter_workspace_size(code, count, rank, adapters)
            work = x.new_empty((size // x.element_size(),))
        st = lib.fpemu_adapter_matmul(
            code, count, k, B.shape[1], rank, adapters, x.data_ptr(), _row_stride(x), A.data_ptr(), A.stride(0),
            A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), None if base is None else base.data_ptr(),
            0 if base is None else base.stride(0), y.data_ptr(), _row_stride(y),
            None if scale.__class__ is float else scale.data_ptr(), scale if scale.__class__ is float else 0.0,
            index.data_ptr(), index.element_size(), plan, None if u is None else u.data_ptr(),
            None if work is None else work.data_ptr(), size, _raw_stream(d))
    if st:
        _lib.check(st, "adapter_matmul")
    _after_call("adapter_matmul", dev)


class _AdapterMatmul(torch.autograd.Function):
    """The operator and its gradients.  Products of the first factor (u) are kept
    for dB; the backward pass makes v = scale * dy B the same way while it makes
    dx, and sums dA and dB over the rows of each adapter."""

    @staticmethod
    def forward(ctx, x, A, B, base, rows, scale):
        y = _packed_like(x if base is None else base, (x.shape[0], B.shape[1]))
        u = torch.empty((x.shape[0], (A.shape[1] + 3) // 4 * 4),
                        dtype=torch.float64 if x.dtype == torch.float64 else torch.float32, device=x.device)
        _launch(x, A, B, base, y, scale, rows, rows.index, u)
        # A tensor of scales is guarded like the others: u holds the values of now.
        ctx.save_for_backward(x, A, B, u, scale if isinstance(scale, torch.Tensor) else None)
        ctx.rows, ctx.scale = rows, scale if scale.__class__ is float else None
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # create_graph: the gradients below are computed outside autograd
            with torch.no_grad():
                *grads, dbase, _, _ = _AdapterMatmul._backward(ctx, dy)
            error = torch._C._functions.DelayedError("adapter_matmul is differentiable once, not twice", 1)
            return *(g if g is None else error(g.requires_grad_(True)) for g in grads), dbase, None, None
        return _AdapterMatmul._backward(ctx, dy)

    @staticmethod
    def _backward(ctx, dy):
        x, A, B, u, scale = ctx.saved_tensors
        if scale is None:
            scale = ctx.scale
        if ctx.rows.capture:
            ctx.rows.check_capture()
        need_x, need_A, need_B, need_base = ctx.needs_input_grad[:4]
        dev = x.device
        d = dev.index
        count = x.shape[0]
        adapters, rank, k = A.shape
        n = B.shape[1]
        dyc = _last_contiguous(dy)
        lib = _lib.load()
        code = _DTYPE_CODE[x.dtype]
        with _on(d):
            dx = _packed_like(x, (count, k)) if need_x else None
            dA = _packed_like(A, (adapters, rank, k)) if need_A else None
            dB = _packed_like(B, (adapters, n, rank)) if need_B else None
            size = v = work = None
            if need_x or need_A:  # v, then the workspace
                size = lib.fpemu_adapter_workspace_size(code, count, rank, adapters)
                v_bytes = u.numel() * u.element_size()  # of rows of 16 bytes or more
                work = x.new_empty(((size + v_bytes) // x.element_size(),))
                v = work.data_ptr()
            st = lib.fpemu_adapter_backward(
                code, count, k, n, rank, adapters, x.data_ptr(), _row_stride(x), A.data_ptr(), A.stride(0), A.stride(1),
                B.data_ptr(), B.stride(0), B.stride(1), dyc.data_ptr(), _row_stride(dyc),
                None if scale.__class__ is float else scale.data_ptr(), scale if scale.__class__ is float else 0.0,
                ctx.rows.plan.data_ptr(), u.data_ptr(), v, None if dx is None else dx.data_ptr(),
                None if dA is None else dA.data_ptr(), None if dB is None else dB.data_ptr(),
                None if v is None else v + v_bytes, size or 0, _raw_stream(d))
        if st:
            _lib.check(st, "adapter_matmul backward")
        _after_call("adapter_matmul backward", dev)
        return dx, dA, dB, dy if need_base else None, None, None


def _span(t):
    first = t.data_ptr()
    return first, first + (sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()


def _check_out(out, shape, x, base, others):
    if out.shape != shape or out.dtype != x.dtype or out.device != x.device:
        raise RuntimeError(f"out must be a {x.dtype} tensor of shape {tuple(shape)} on {x.device}")
    o2 = out.view(-1, shape[-1]) if out.numel() else out.reshape(math.prod(shape[:-1]), shape[-1])
    if out.numel() == 0:
        return o2
    if o2.stride(-1) != 1 and o2.shape[-1] > 1 or o2.shape[0] > 1 and o2.stride(0) < o2.shape[1]:
        raise RuntimeError("out needs a contiguous last dimension and rows that do not overlap")
    lo, hi = _span(o2)
    for t in others:
        if t.numel():
            a, b = _span(t)
            if a < hi and lo < b:
                raise RuntimeError("out overlaps an input")
    if base is not None:
        a, b = _span(base)
        if a < hi and lo < b and not (base.data_ptr() == out.data_ptr() and base.shape == out.shape
                                      and base.stride() == out.stride()):
            raise RuntimeError("out overlaps base without being base")
    return o2


def adapter_matmul(x, A, B, rows, base=None, scale=1.0, out=None):
    """``base + scale_i * (x @ A[i].T) @ B[i].T`` with each row's own adapter i.

    x: [..., k]; A: [adapters, rank, k]; B: [adapters, n, rank], all of one float
    dtype (float64, float32, float16, bfloat16).  rows: ``prepare_rows(...)`` of
    the batch (of x's leading shape, unless one of the two is flat), or an int32/int64
    tensor of ids whose shape is x's leading shape or the first dimensions of it (-1: no
    adapter; such a row returns ``base``).
    base: broadcastable to [..., n], or None for zero.  scale: one number, or a
    tensor with one value for each adapter (no gradient; like the other operands it
    must not change in place before the backward pass).  out: where to write the
    result when autograd does not record; it may be ``base`` itself.

    Sums are held in float64 for float64 and in float32 otherwise, and the result is
    rounded once.  Before that: a product of float32 values is made of tensor-core parts
    and off by 2^-21 of it at most; sums of up to 64 tensor-core instructions are
    truncated, not rounded (5e-6 of a long sum of one sign; 7e-7 for float32); with
    float16 the intermediate ``x @ A[i].T`` enters the second product with 22 bits
    (values below 2^-17 of their row's largest with fewer), with bfloat16 with all 24.
    x, A, B and base have gradients (once; not twice differentiable, and not in forward
    mode); repeated calls give the same bits."""
    dtype = x.dtype
    _dtype_bits(dtype)
    _no_tangents("adapter_matmul", x, A, B, base, scale)
    d = x.get_device()
    if d < 0 or A.get_device() != d or B.get_device() != d or (base is not None and base.get_device() != d) \
            or d not in _lib._watched:
        _require_cuda(x, A, B, *(() if base is None else (base,)))
    if A.dtype is not dtype or B.dtype is not dtype or (base is not None and base.dtype is not dtype):
        raise TypeError("adapter_matmul: operands of one dtype, got " +
                        ", ".join(str(t.dtype) for t in (x, A, B, base) if t is not None))
    shape_x, shape_A, shape_B = x.shape, A.shape, B.shape
    if len(shape_x) < 1 or len(shape_A) != 3 or len(shape_B) != 3 or shape_A[0] != shape_B[0] \
            or shape_A[1] != shape_B[2] or shape_A[2] != shape_x[-1]:
        raise RuntimeError(f"adapter_matmul: expected x [..., k], A [adapters, rank, k], B [adapters, n, rank], got "
                           f"{tuple(shape_x)}, {tuple(shape_A)}, {tuple(shape_B)}")
    adapters, rank, k = shape_A
    n = shape_B[1]
    if not 1 <= rank <= _lib.FPEMU_ADAPTER_MAX_RANK:
        raise ValueError(f"adapter_matmul: rank {rank}; between 1 and {_lib.FPEMU_ADAPTER_MAX_RANK} is supported")
    if not 1 <= adapters <= _lib.FPEMU_ADAPTER_MAX_COUNT:
        raise ValueError(f"adapter_matmul: {adapters} adapters; between 1 and {_lib.FPEMU_ADAPTER_MAX_COUNT}")
    if isinstance(scale, torch.Tensor):
        if scale.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("adapter_matmul: scale has no gradient")
        if scale.shape != (adapters,):
            raise RuntimeError(f"adapter_matmul: scale of shape {tuple(scale.shape)} for {adapters} adapters")
        if scale.dtype is not torch.float64 or scale.get_device() != d or not scale.is_contiguous():
            scale = scale.detach().to(device=x.device, dtype=torch.float64).contiguous()
    else:
        scale = float(scale)
    flat = len(shape_x) == 2
    lead = shape_x[:-1]
    count = shape_x[0] if flat else math.prod(lead)
    shape = lead + (n,)
    records = torch.is_grad_enabled() and (x.requires_grad or A.requires_grad or B.requires_grad
                                           or (base is not None and base.requires_grad))
    if isinstance(rows, PreparedRows):
        if rows.adapters != adapters:
            raise RuntimeError(f"adapter_matmul: rows prepared for {rows.adapters} adapters, not {adapters}")
        index = rows.index
        if index.shape[0] != count:
            raise RuntimeError(f"adapter_matmul: {index.shape[0]} prepared rows for {count} rows of x")
        if rows.shape != lead and len(rows.shape) > 1 and not flat:
            raise RuntimeError(f"adapter_matmul: rows prepared for {tuple(rows.shape)}, x has rows of {tuple(lead)}")
        if index.get_device() != d:
            raise RuntimeError(f"operands on different devices: {x.device} and {index.device}")
        if rows.capture:
            rows.check_capture()
    elif isinstance(rows, torch.Tensor):
        if rows.dtype not in (torch.int32, torch.int64):
            raise TypeError("adapter ids are an int32 or int64 tensor")
        if rows.get_device() != d:
            _require_cuda(x, rows)
        index = _spread_index(rows, lead)
        if records or count > _lib.FPEMU_ADAPTER_FEW_ROWS:
            rows = PreparedRows(index, adapters)
        else:
            rows = None
            index = index.reshape(-1).contiguous()
    else:
        raise TypeError("rows is a tensor of adapter ids or the result of prepare_rows")
    x2, A, B = _last_contiguous(x if flat else x.reshape(count, k)), _last_contiguous(A), _last_contiguous(B)
    base2 = None
    if base is not None:
        if base.shape != shape:
            base = base.expand(shape)
        base2 = _last_contiguous(base if flat else base.reshape(count, n))
    if records:
        if out is not None:
            raise RuntimeError("adapter_matmul: out cannot be given while autograd records")
        y = _AdapterMatmul.apply(x2, A, B, base2, rows, scale)
        return y if flat else y.view(shape)
    if out is None:
        y = _packed_like(x2 if base2 is None else base2, (count, n))
    else:
        if out.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("adapter_matmul: out requires a gradient, which would not include this call")
        y = _check_out(out, shape, x, base, (x2, A, B, index) + ((scale,) if scale.__class__ is not float else ()))
    _launch(x2, A, B, base2, y, scale, rows, index, None)
    if out is None:
        return y if flat else y.view(shape)
    torch.autograd.graph.increment_version(out)
    return out


class Adapters(nn.Module):
    """The factors of ``adapters`` low-rank adapters of one projection: A
    [adapters, rank, in_features] and B [adapters, out_features, rank], with B zero
    at first so that a new adapter changes nothing.  ``scale`` is alpha / rank."""

    def __init__(self, adapters, in_features, out_features, rank, alpha=None, device=None, dtype=torch.float64):
        super().__init__()
        _dtype_bits(dtype)
        if not 1 <= rank <= _lib.FPEMU_ADAPTER_MAX_RANK:
            raise ValueError(f"rank {rank}; between 1 and {_lib.FPEMU_ADAPTER_MAX_RANK} is supported")
        self.scale = (rank if alpha is None else alpha) / rank
        self.A = nn.Parameter(torch.empty((adapters, rank, in_features), device=device, dtype=dtype))
        self.B = nn.Parameter(torch.zeros((adapters, out_features, rank), device=device, dtype=dtype))
        bound = 1.0 / math.sqrt(max(in_features, 1))
        nn.init.uniform_(self.A, -bound, bound)

    @property
    def adapters(self):
        return self.A.shape[0]

    def extra_repr(self):
        n, rank, k = self.A.shape
        return f"adapters={n}, in_features={k}, out_features={self.B.shape[1]}, rank={rank}, scale={self.scale}"

    def forward(self, x, rows, base=None, out=None):
        return adapter_matmul(x, self.A, self.B, rows, base=base, scale=self.scale, out=out)


_captured_ids = weakref.WeakKeyDictionary()  # model -> the ids that graphs captured in its blocks read


class _ActiveRows:
    """The ids of the batch inside a ``use_adapters`` block; grouped once for each
    leading shape that the layers meet on a stream.  Streams are not ordered among
    each other, and what a capture makes is there after a replay alone: each stream,
    and each capture, has plans of its own."""

    def __init__(self, index, model=None):
        self.index = index.clone()
        self.prepared = {}
        self.lock = threading.Lock()
        self.kept = [] if model is None else _captured_ids.setdefault(model, [])
        d = index.get_device()
        if d >= 0:  # else the first layer refuses it
            self.stream, self.capture = _raw_stream(d), _capture_id(d)
            self.copied = torch.cuda.Event()
            self.copied.record(torch.cuda.current_stream(d))

    def __reduce__(self):
        """A copy of a model (or a pickled one) inside the block has the block's ids, and groups them anew."""
        return _ActiveRows, (self.index,)

    def prepare(self, lead, adapters):
        d = self.index.get_device()
        if d < 0:
            return PreparedRows(self.index, adapters, lead)
        stream, capture = _raw_stream(d), _capture_id(d)
        if self.capture and capture != self.capture:
            raise RuntimeError("a use_adapters block that began in the capture of a CUDA graph serves that capture alone")
        key = (tuple(lead), adapters, stream, capture)
        with self.lock:
            if key not in self.prepared:
                if stream != self.stream:
                    current = torch.cuda.current_stream(d)
                    if capture == self.capture:  # a capture cannot wait for what was issued before it
                        current.wait_event(self.copied)
                    self.index.record_stream(current)
                if capture != self.capture:  # the graph copies the ids at every replay, after the block too
                    self.kept.append(self.index)
                self.prepared[key] = PreparedRows(self.index, adapters, lead)
            return self.prepared[key]


@contextlib.contextmanager
def use_adapters(model, index):
    """Within the block, the model's layers that have adapters (``add_adapters``)
    apply row t's adapter ``index[t]`` (-1: none).  ``index`` has the leading shape
    of the layers' inputs, or the first dimensions of it, and is copied as the block
    begins: later changes of it take no effect (a CUDA graph that is to follow them
    captures the whole block; one captured inside keeps the block's ids).  The block
    holds for the model, in every thread and on every stream, but one that begins in a
    capture serves that capture alone.  A backward pass that computes the layers again
    (activation checkpointing) has to run inside it."""
    from fp_emulation.nn import Linear

    if not isinstance(index, torch.Tensor) or index.dtype not in (torch.int32, torch.int64):
        raise TypeError("adapter ids are an int32 or int64 tensor")

    layers = [m for m in model.modules() if isinstance(m, Linear) and m._modules.get("adapters") is not None]
    if not layers:
        raise RuntimeError("use_adapters: the model has no Linear with adapters (add_adapters)")
    before = [m.active_rows for m in layers]
    active = _ActiveRows(index, model)
    for m in layers:
        m.active_rows = active
    try:
        yield model
    finally:
        for m, rows in zip(layers, before):
            m.active_rows = rows


def add_adapters(model, adapters, rank, alpha=None):
    """Put ``adapters`` low-rank adapters beside every ``fp_emulation.Linear`` of
    ``model`` (as ``layer.adapters``, float64 like the layer) and return the model.
    Outside a ``use_adapters`` block the layers compute as before."""
    from fp_emulation.nn import Linear

    for m in list(model.modules()):
        if isinstance(m, Linear):
            m.adapters = Adapters(adapters, m.in_features, m.out_features, rank, alpha, device=m.weight.device)
    return model
