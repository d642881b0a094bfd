"""grad_norm and clip_grads over a tensor of more than 2^31 elements."""
from __future__ import annotations

import math

import pytest
import torch

import fp_emulation as fp

pytestmark = pytest.mark.gpu


def test_offsets_past_32_bits():
    n = 2 ** 31 + 1003
    g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g[-1], g[-2] = 65536, -131072
    total = math.sqrt(n - 2 + 2.0 ** 32 + 2.0 ** 34)
    small = torch.full((5,), 3.0, dtype=torch.float64, device="cuda")
    want = math.sqrt(total ** 2 + 45)
    out, norm = fp.clip_grads([g, small], 1.0)
    # the sums are of integers below 2^53; the root and its square here round a few times
    assert norm.dtype == torch.float64 and abs(norm.item() - want) <= 4 * 2.0 ** -53 * want
    c = 1.0 / (want + 1e-6)
    for i in (0, 2 ** 31 - 1, 2 ** 31, n - 3, n - 2, n - 1):
        assert out[0][i].item() == pytest.approx(g[i].item() * c, rel=2 ** -8 * 1.01)
    assert (out[0][:-2] == out[0][0]).all()
    assert fp.grad_norm([g], math.inf).item() == 131072
    assert fp.grad_norm(g, 1).item() == pytest.approx(n - 2 + 65536 + 131072, rel=2 ** -24)
