"""Long batches whose slots (up to 64 rows of one adapter) pass quickly: one to three
chunks each, of 1 to 64 rows, so that the warps of a block are often several slots
apart.  What one slot leaves in shared memory may not reach the next one's results:
the formula in float64 (tolerances of test_gpu_adapters), and the same bits every
time."""
from __future__ import annotations

import pytest
import torch

import fp_emulation as fp
from test_gpu_adapters import DTYPES, _close, _data

pytestmark = pytest.mark.gpu

# k and n of one chunk, two, and three (a chunk is 16 doubles, 32 floats, 64 16-bit values)
WIDTHS = {torch.float64: [(2, 16), (20, 1), (48, 40)], torch.float32: [(2, 32), (40, 1), (96, 80)],
          torch.float16: [(2, 64), (80, 1), (192, 160)], torch.bfloat16: [(2, 64), (80, 1), (192, 160)]}


def _uneven(n, rows, gen):
    """Adapters of 1, 2, ... 64, 65, ... rows in turn, in random order, some rows without one."""
    counts = torch.arange(n) % 130 + 1
    ids = torch.repeat_interleave(torch.arange(n), counts)[:rows]
    ids = torch.cat([ids, torch.full((rows - len(ids),), -1)])
    return ids[torch.randperm(rows, generator=gen)].to(torch.int32).cuda()


def _by_rows(x, A, B, scale, index):
    """s B (A x) of every row with its own factors, the magnitudes of its sums, u and its own."""
    out = [[], [], [], []]
    for a in range(0, x.shape[0], 1000):
        i = index[a:a + 1000].long()
        on = ((i >= 0) * scale[i.clamp(min=0)])[:, None]
        xs, As, Bs = x[a:a + 1000].double(), A[i.clamp(min=0)].double(), B[i.clamp(min=0)].double()
        u = on * torch.einsum("trk,tk->tr", As, xs)
        ua = on * torch.einsum("trk,tk->tr", As.abs(), xs.abs())
        for o, v in zip(out, (torch.einsum("tnr,tr->tn", Bs, u), torch.einsum("tnr,tr->tn", Bs.abs(), ua), u, ua)):
            o.append(v)
    return [torch.cat(o) for o in out]


@pytest.mark.parametrize("r", [16, 40, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_one_slot_does_not_reach_the_next(dtype, r):
    for seed, (k, m) in enumerate(WIDTHS[dtype]):
        n, rows = 200, 13000
        x, A, B, base, dy, scale, _ = _data(rows, n, k, m, r, dtype, seed=seed)
        index = _uneven(n, rows, torch.Generator().manual_seed(seed))
        for t in (x, A, B):
            t.requires_grad_(True)
        plan = fp.prepare_rows(index, n)

        def step():
            y = fp.adapter_matmul(x, A, B, plan, base=base, scale=scale)
            return (y.detach(), *torch.autograd.grad(y, (x, A, B), dy))

        first = step()
        with torch.no_grad():
            y, mag, u, ua = _by_rows(x, A, B, scale, index)
            _close(first[0], base.double() + y, base.double().abs() + mag, k + r, dtype)
            dx, dxm, v, va = _by_rows(dy, B.transpose(1, 2), A.transpose(1, 2), scale, index)
            _close(first[1], dx, dxm, m + r, dtype)
            for i in (0, 1, 63, 64, 127, n - 1):
                t = index == i
                _close(first[2][i], v[t].T @ x[t].double(), va[t].T @ x[t].double().abs(), m + rows, dtype)
                _close(first[3][i], dy[t].double().T @ u[t], dy[t].double().abs().T @ ua[t], k + rows, dtype)
            for _ in range(20):
                assert torch.equal(fp.adapter_matmul(x, A, B, plan, base=base, scale=scale), first[0])
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(step(), first))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_in_runs_beside_rows_in_any_order(dtype):
    """Slots whose rows follow one another (copied in one box) and slots whose rows do not (copied
    one by one) share the buffers in turn; x and base of odd strides, never copied in boxes, give
    the same bits."""
    n, rows, k, m, r = 60, 9000, 256, 320, 16
    x, A, B, base, dy, scale, _ = _data(rows, n, k, m, r, dtype)
    index = torch.arange(rows, device="cuda") * n // rows
    gen = torch.Generator(device="cuda").manual_seed(2)
    loose = torch.nonzero(index % 2).flatten()  # every other adapter's rows change places among themselves
    index[loose] = index[loose[torch.randperm(len(loose), generator=gen, device="cuda")]]

    def odd(t):
        view = torch.zeros((rows, t.shape[1] + 1), dtype=dtype, device="cuda")[:, :t.shape[1]]
        view.copy_(t)
        return view

    plan = fp.prepare_rows(index, n)
    want = fp.adapter_matmul(odd(x), A, B, plan, base=odd(base), scale=scale)
    for _ in range(20):
        assert torch.equal(fp.adapter_matmul(x, A, B, plan, base=base, scale=scale), want)
