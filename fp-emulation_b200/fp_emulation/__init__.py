"""fp_emulation -- B200 (sm_100a) build of Ozaki scheme II FP64 emulation.

Drop-in for the reference package's GEMM path (its ``__init__.py:1-13``):
``ozaki2_int8_matmul``, ``Linear`` and ``convert``.  The reference's ML-PLAC
helpers (fit_pwl, eval_pwl, ...) are not part of this build.  Beside it, for
training and serving converted models: low-rank adapters of many requests
(``adapter_matmul``, ``prepare_rows``, ``Adapters``, ``add_adapters``,
``use_adapters``) and the global gradient norm (``grad_norm``, ``clip_grads``,
``clip_grad_norm_``).
"""
from fp_emulation.adapters import Adapters, PreparedRows, adapter_matmul, add_adapters, prepare_rows, use_adapters
from fp_emulation.gradients import clip_grad_norm_, clip_grads, grad_norm
from fp_emulation.nn import Linear, convert
from fp_emulation.ozaki import PreparedOperand, ozaki2_int8_matmul, prepare_operand

__all__ = ["Linear", "convert", "ozaki2_int8_matmul", "PreparedOperand", "prepare_operand",
           "Adapters", "PreparedRows", "adapter_matmul", "add_adapters", "prepare_rows", "use_adapters",
           "clip_grad_norm_", "clip_grads", "grad_norm"]
