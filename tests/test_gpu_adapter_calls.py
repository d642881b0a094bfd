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
