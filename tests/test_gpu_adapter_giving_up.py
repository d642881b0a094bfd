"""Adapter kernels whose copies stall between and within slots of one to three chunks,
in training, without a GPU fault (the test hook of test_gpu_adapter_failure).  Whichever
warp's wait runs out first, the blocks end, and each value of the results and of the
gradients made from them is NaN or the one an undisturbed call gives."""
from __future__ import annotations

import os
import traceback

import pytest

pytestmark = pytest.mark.gpu


def _child(dtype, q):
    try:
        os.environ["FPEMU_WAIT_BUDGET_MS"] = "50"
        import torch

        import fp_emulation as fp
        from fp_emulation import _lib, ozaki

        ozaki._CHECK_MODE = "off"
        out = []
        gen = torch.Generator(device="cuda").manual_seed(1)
        for k, m in ((40, 24), (24, 160)):
            rows, n, r = 30000, 400, 12

            def rnd(*shape):
                return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64).to(getattr(torch, dtype))

            x, A, B, base, dy = rnd(rows, k), rnd(n, r, k), rnd(n, m, r), rnd(rows, m), rnd(rows, m)
            for t in (x, A, B):
                t.requires_grad_(True)
            plan = fp.prepare_rows(torch.randint(-1, n, (rows,), generator=gen, device="cuda"), n)

            def step(forward=None, backward=None):
                for unit, call in ((forward, lambda: fp.adapter_matmul(x, A, B, plan, base=base)),
                                   (backward, lambda: torch.autograd.grad(y, (x, A, B), dy))):
                    if unit is not None:
                        os.environ["FPEMU_TEST_STALL_UNIT"] = str(unit)
                    got = call()
                    os.environ.pop("FPEMU_TEST_STALL_UNIT", None)
                    if torch.is_tensor(got):
                        y = got
                torch.cuda.synchronize()
                return (y.detach(), *got)

            want = step()
            assert _lib.device_error(clear=True)[0] == 0
            for unit in range(5):
                for which in ("forward", "backward"):
                    got = step(**{which: unit})
                    error = _lib.device_error(clear=True)[:2]
                    lost = [torch.isnan(g) for g in got]
                    out.append((error, [int(b.sum()) for b in lost],
                                all(torch.equal(g[~b], w[~b]) for g, b, w in zip(got, lost, want))))
            again = step()
            assert _lib.device_error(clear=True)[0] == 0 and all(torch.equal(a, b) for a, b in zip(again, want))
        q.put(("ok", out))
    except Exception:
        q.put(("error", traceback.format_exc()))


@pytest.mark.parametrize("dtype", ["float64", "float32", "float16", "bfloat16"])
def test_every_value_is_right_or_nan(dtype):
    import torch.multiprocessing as mp

    from fp_emulation import _lib

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_child, args=(dtype, q))
    p.start()
    status, out = q.get(timeout=240)
    p.join(timeout=60)
    assert status == "ok", out
    for (error, where), lost, rest in out:
        assert rest, "a value that is not NaN is the undisturbed one"
        assert (error == _lib.FPEMU_ERR_TIMEOUT and where in (17, 18)) == any(lost)
    assert any(lost[0] for _, lost, _ in out) and any(lost[3] for _, lost, _ in out), "something did stall"
