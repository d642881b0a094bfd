"""The global norm of many gradients, and clipping by it.

A converted model mixes float64 layers with whatever the rest of the model is
made of; the norm here goes over tensors of any float dtypes and sizes at once,
with every sum held in float64.  CUDA tensors only.  ``clip_grad_norm_`` keeps the
signature of ``torch.nn.utils.clip_grad_norm_``; nothing here has a counterpart in
the reference.
"""
from __future__ import annotations

import math
import operator
from array import array

import torch

from fp_emulation import _lib
from fp_emulation.adapters import _DTYPE_CODE, _no_tangents
from fp_emulation.ozaki import _after_call, _dtype_bits, _on, _raw_stream, _require_cuda

_NORMS = {1.0: 1, 2.0: 2, math.inf: 0}


def _norm_code(norm_type):
    try:
        return _NORMS[float(norm_type)]
    except KeyError:
        raise ValueError(f"norm_type {norm_type}: 1, 2 and inf are supported") from None


def _dense(t):
    """Whether t's elements fill one stretch of memory, each once, in any order."""
    if t.is_contiguous():
        return True
    need = 1
    for stride, size in sorted((st, s) for s, st in zip(t.shape, t.stride()) if s != 1):
        if stride != need:
            return False
        need *= size
    return True


_layout, _dtype, _grad = map(operator.attrgetter, ("layout", "dtype", "grad"))


def _check_list(tensors, what):
    """The tensors' dtype codes; refuses what the kernels do not take."""
    _no_tangents(what, *tensors)
    try:
        devices = set(map(torch.Tensor.get_device, tensors))
        codes = list(map(_DTYPE_CODE.__getitem__, map(_dtype, tensors)))
        if len(devices) == 1 and devices <= _lib._watched and set(map(_layout, tensors)) == {torch.strided}:
            return codes
    except (TypeError, KeyError):
        pass
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: a list of tensors, got {type(t).__name__}")
        if t.layout is not torch.strided:
            raise TypeError(f"{what}: strided tensors only, got {t.layout}")
        _dtype_bits(t.dtype)
    _require_cuda(*tensors)
    return [_DTYPE_CODE[t.dtype] for t in tensors]


def _in_one_stretch(tensors):
    """The tensors, with copies in place of those that are not dense."""
    if all(map(torch.Tensor.is_contiguous, tensors)):
        return tensors
    return [t if _dense(t) else t.contiguous() for t in tensors]


def _run(src, dst, codes, norm_code, max_norm, what):
    """One fpemu_clip_grads: the norm of `src` and, with `dst`, the scaled tensors.
    The norm is float64 if any tensor is, else float32."""
    n = len(src)
    dev = src[0].device
    wide = _lib.FPEMU_DT_F64 in codes
    lib = _lib.load()
    ptrs, sizes = array("Q", map(torch.Tensor.data_ptr, src)), array("q", map(torch.Tensor.numel, src))
    outs = None if dst is None else ptrs if dst is src else array("Q", map(torch.Tensor.data_ptr, dst))
    kinds = array("i", codes)
    with _on(dev.index):
        norm = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=dev)
        ws = torch.empty((lib.fpemu_clip_workspace_size(n),), dtype=torch.uint8, device=dev)
        st = lib.fpemu_clip_grads(n, ptrs.buffer_info()[0], None if outs is None else outs.buffer_info()[0],
                                  sizes.buffer_info()[0], kinds.buffer_info()[0], norm_code, max_norm,
                                  norm.data_ptr(), int(wide), ws.data_ptr(), ws.numel(),
                                  _raw_stream(dev.index))
    if st:
        _lib.check(st, what)
    _after_call(what, dev)
    return norm


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm {max_norm}: a number >= 0")
    return max_norm


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """The norm (1, 2 or inf) over every element of every tensor, as a 0-d tensor
    on their device: float64 if one of them is float64, else float32.  Sums are
    held in float64, and squares neither overflow nor vanish before the norm does.
    The result has no gradient.  No tensors: 0 on the CPU."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    if not tensors:
        return torch.tensor(0.0)
    codes = _check_list(tensors, "grad_norm")
    return _run(_in_one_stretch(tensors), None, codes, code, 0.0, "grad_norm")


@torch.no_grad()
def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """``(clipped, norm)``: new tensors, the gradients times
    ``min(1, max_norm / (norm + 1e-6))``, and their global norm before.  The
    gradients stay as they are (those of ``torch.autograd.grad``, say); the results have
    none of their own.  out: tensors
    to write to, of the gradients' shapes and dtypes; none may overlap another
    tensor, but each may be its own gradient."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    code, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    if not grads:
        return [], torch.tensor(0.0)
    codes = _check_list(grads, "clip_grads")
    src = _in_one_stretch(grads)
    if out is None:
        out = dst = [torch.empty_like(s) for s in src]
        return out, _run(src, dst, codes, code, max_norm, "clip_grads")
    out = list(out)
    if len(out) != len(grads):
        raise RuntimeError(f"clip_grads: {len(out)} outputs for {len(grads)} gradients")
    if all(map(operator.is_, out, src)):
        norm = _run(src, src, codes, code, max_norm, "clip_grads")
        torch.autograd.graph.increment_version(out)
        return out, norm
    _check_list(grads + out, "clip_grads")
    for g, o in zip(grads, out):
        if g.shape != o.shape or g.dtype != o.dtype:
            raise RuntimeError("clip_grads: an output has another shape or dtype than its gradient")
    dst = [o if _dense(o) and o.stride() == s.stride() else torch.empty_like(s) for s, o in zip(src, out)]
    norm = _run(src, dst, codes, code, max_norm, "clip_grads")
    torch.autograd.graph.increment_version([o for o, d in zip(out, dst) if o is d])
    for o, d in zip(out, dst):
        if o is not d:
            o.copy_(d)
    return out, norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """Scale the gradients of ``parameters`` in place to a global norm of at most
    ``max_norm`` and return the norm before (see ``grad_norm``); parameters without
    a gradient are passed over.  With ``error_if_nonfinite`` the norm is read back
    first, and a RuntimeError leaves the gradients as they were.  Each gradient may
    appear once.  ``foreach`` is there for callers of the other: all tensors go at once."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    code, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    grads = [g for g in map(_grad, parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is "
                               f"non-finite ({norm.item()}), so it cannot be clipped")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]
