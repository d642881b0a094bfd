"""A wait of the adapter kernels that runs out, without a GPU fault.

The test hook FPEMU_TEST_STALL_UNIT makes the copying warps of each kernel's first
block stop after that many chunks, as stalled copies would; the computing warps
give up after FPEMU_WAIT_BUDGET_MS, record FPEMU_ERR_TIMEOUT, turn what they could
not finish into NaN and unwind.  A fresh process each, since the budget is read once."""
from __future__ import annotations

import os
import traceback

import pytest

pytestmark = pytest.mark.gpu


def _child(dtype, unit, q):
    try:
        os.environ["FPEMU_WAIT_BUDGET_MS"] = "100"
        os.environ.pop("FPEMU_CHECK", None)
        import torch

        import fp_emulation as fp
        from fp_emulation import _lib

        gen = torch.Generator(device="cuda").manual_seed(1)
        rows, n, k, m, r = 2000, 3, 520, 712, 8

        def rnd(*shape):
            return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64).to(getattr(torch, dtype))

        x, A, B, base = rnd(rows, k), rnd(n, r, k), rnd(n, m, r), rnd(rows, m)
        index = torch.sort(torch.randint(n, (rows,), generator=gen, device="cuda"))[0]
        plan = fp.prepare_rows(index, n)
        want = fp.adapter_matmul(x, A, B, plan, base=base)
        torch.cuda.synchronize()
        os.environ["FPEMU_TEST_STALL_UNIT"] = str(unit)
        out = {}
        try:
            got = fp.adapter_matmul(x, A, B, plan, base=base)
        except _lib.FpemuError:
            got = None
        torch.cuda.synchronize()
        os.environ.pop("FPEMU_TEST_STALL_UNIT")
        out["poll"] = _lib.poll_error()
        if got is not None:
            nan = torch.isnan(got)
            out["nan"], out["rest"] = int(nan.sum()), bool(torch.equal(got[~nan], want[~nan]))
        try:
            fp.adapter_matmul(x, A, B, plan, base=base)
            out["raised"] = None
        except _lib.FpemuError as exc:
            out["raised"] = exc.status
        torch.cuda.synchronize()
        out["again"] = bool(torch.equal(fp.adapter_matmul(x, A, B, plan, base=base), want))
        torch.cuda.synchronize()
        out["after"] = _lib.device_error(clear=True)[0]
        q.put(("ok", out))
    except Exception:
        q.put(("error", traceback.format_exc()))


@pytest.mark.parametrize("unit", [0, 1])
@pytest.mark.parametrize("dtype", ["float64", "bfloat16"])
def test_a_stalled_chunk_shows_as_nan_and_raises(dtype, unit):
    import torch.multiprocessing as mp

    from fp_emulation import _lib

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_child, args=(dtype, unit, q))
    p.start()
    status, out = q.get(timeout=240)
    p.join(timeout=60)
    assert status == "ok", out
    if "nan" in out:  # the call returned before its kernel gave up
        assert out["poll"][0] == _lib.FPEMU_ERR_TIMEOUT and out["poll"][1] in (17, 18)
        assert out["nan"] > 0 and out["rest"], "what was finished is exact, what was not is NaN"
        assert out["raised"] == _lib.FPEMU_ERR_TIMEOUT
    assert out["again"] and out["after"] == 0
