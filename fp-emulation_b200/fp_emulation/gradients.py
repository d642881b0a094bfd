"""The global norm of many gradients, and clipping by it.

A converted model mixes float64 layers with whatever the rest of the model is
made of; the norm here goes over tensors of any float dtypes and sizes at once,
with every sum held in float64.  CUDA tensors only.  ``clip_grad_norm_`` keeps the
signature of ``torch.nn.utils.clip_grad_norm_``; nothing here has a counterpart in
the reference.
"""
from __future__ import annotations

import ctypes
import math

import torch

from fp_emulation import _lib
from fp_emulation.adapters import _DTYPE_CODE
from fp_emulation.ozaki import _after_call, _dtype_bits, _require_cuda, _stream

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


def _check_list(tensors, what):
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: a list of tensors, got {type(t).__name__}")
        if t.layout != torch.strided:
            raise TypeError(f"{what}: strided tensors only, got {t.layout}")
        if t.dtype not in _DTYPE_CODE:
            _dtype_bits(t.dtype)  # raises
    return _require_cuda(*tensors)


def _run(src, dst, code, max_norm, dev, what):
    """One fpemu_clip_grads: the norm of `src` and, with `dst`, the scaled tensors.
    float64 if any tensor is, else float32."""
    n = len(src)
    wide = any(t.dtype == torch.float64 for t in src)
    lib = _lib.load()
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in src])
    outs = None if dst is None else (ctypes.c_void_p * n)(*[t.data_ptr() for t in dst])
    sizes = (ctypes.c_int64 * n)(*[t.numel() for t in src])
    dtypes = (ctypes.c_int32 * n)(*[_DTYPE_CODE[t.dtype] for t in src])
    with torch.cuda.device(dev):
        norm = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=dev)
        ws = torch.empty((lib.fpemu_clip_workspace_size(n),), dtype=torch.uint8, device=dev)
        st = lib.fpemu_clip_grads(n, ptrs, outs, sizes, dtypes, code, max_norm, norm.data_ptr(), int(wide),
                                  ws.data_ptr(), ws.numel(), _stream(dev))
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
    No tensors: 0 on the CPU."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    if not tensors:
        return torch.tensor(0.0)
    dev = _check_list(tensors, "grad_norm")
    return _run([t if _dense(t) else t.contiguous() for t in tensors], None, code, 0.0, dev, "grad_norm")


@torch.no_grad()
def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """``(clipped, norm)``: new tensors, the gradients times
    ``min(1, max_norm / (norm + 1e-6))``, and their global norm before.  The
    gradients stay as they are (those of ``torch.autograd.grad``, say).  out: tensors
    to write to, of the gradients' shapes and dtypes; none may overlap another
    tensor, but each may be its own gradient."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    code, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    if not grads:
        return [], torch.tensor(0.0)
    dev = _check_list(grads, "clip_grads")
    src = [g if _dense(g) else g.contiguous() for g in grads]
    if out is None:
        out = dst = [torch.empty_like(s) for s in src]
    else:
        out = list(out)
        if len(out) != len(grads):
            raise RuntimeError(f"clip_grads: {len(out)} outputs for {len(grads)} gradients")
        _check_list(grads + out, "clip_grads")
        for g, o in zip(grads, out):
            if g.shape != o.shape or g.dtype != o.dtype:
                raise RuntimeError("clip_grads: an output has another shape or dtype than its gradient")
        dst = [o if _dense(o) and o.stride() == s.stride() else torch.empty_like(s) for s, o in zip(src, out)]
    norm = _run(src, dst, code, max_norm, dev, "clip_grads")
    if dst is not out:
        for o, d in zip(out, dst):
            if o is d:
                torch.autograd.graph.increment_version(o)
            else:
                o.copy_(d)
    return out, norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scale the gradients of ``parameters`` in place to a global norm of at most
    ``max_norm`` and return the norm before (see ``grad_norm``); parameters without
    a gradient are passed over.  With ``error_if_nonfinite`` the norm is read back
    first, and a RuntimeError leaves the gradients as they were.  Each gradient may
    appear once."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    code, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is "
                               f"non-finite ({norm.item()}), so it cannot be clipped")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]
