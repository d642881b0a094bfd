"""Clipping whose factor is far below the range of a float: gradients and limits that
lie far apart, float64 tensors beside narrower ones.  Tolerances of test_gpu_clip."""
from __future__ import annotations

import math

import pytest
import torch

import fp_emulation as fp
from test_gpu_clip import _check_scaled, _exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [29, 31, 37, 38, 40, 44, 45, 46, 60])
def test_narrow_gradients_beside_a_far_norm(exponent):
    gen = torch.Generator(device="cuda").manual_seed(exponent)

    def rand(n):
        return torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) + 0.5

    # the last ones end among bfloat16's and float's own subnormal numbers, or at 0
    for size in (1e30, 1e10, 1.0):
        grads = [rand(1000) * 10.0 ** exponent, (rand(5001) * size).float(), (rand(3003) * size).bfloat16(),
                 rand(777).half()]
        norm = _exact(grads, 2)
        out, got = fp.clip_grads(grads, 1.0)
        assert abs(got.item() - norm) <= 2.0 ** -45 * norm
        _check_scaled(out, grads, 1.0 / (norm + 1e-6))
        fp.clip_grads(grads, 1.0, out=grads)
        assert all(torch.equal(a, b) for a, b in zip(grads, out))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_norm_past_the_largest_float(dtype):
    g = torch.full((10007,), 3e38, dtype=torch.float64, device="cuda").to(dtype)
    g[1::3] = 2e38
    norm = _exact([g], 2)
    out, got = fp.clip_grads([g], 1.0)
    assert math.isinf(got.item())  # the norm is a float; the factor is made from the double
    _check_scaled(out, [g], 1.0 / (norm + 1e-6))
    far = torch.full((5,), 1e30, dtype=dtype, device="cuda")
    out, _ = fp.clip_grads([far], 1e-10)  # the norm is in range, the factor is 4e-41
    _check_scaled(out, [far], 1e-10 / (_exact([far], 2) + 1e-6))
