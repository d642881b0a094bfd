"""adapter_matmul, its gradients and the Linear layers' adapters on the GPU,
against the formulas in float64.

Tolerances, elementwise: a sum of K products held with unit e is off by at most
(K + 2) e times the sum of the products' magnitudes, whatever the order, and the
result is rounded once (half a step of its type).  e is 2^-53 for float64 and
2^-23 otherwise (2^-24, doubled for adders that truncate).  16-bit data may hold
the rank-long intermediate as two 16-bit parts: 2^-15 of its magnitude."""
from __future__ import annotations

import pytest
import torch

import fp_emulation as fp
from fp_emulation import _lib

pytestmark = pytest.mark.gpu

DTYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]
# rows, adapters, k, n, rank
SIZES = [(1, 1, 1, 1, 1), (1, 5, 7, 3, 2), (5, 3, 33, 17, 8), (64, 4, 256, 256, 16), (256, 300, 40, 24, 4),
         (257, 7, 130, 65, 12), (300, 1, 64, 64, 128), (700, 9, 1000, 777, 33), (65, 2, 16, 4100, 64),
         (1025, 5, 512, 96, 16), (3000, 3, 72, 1032, 40), (40, 2, 4096, 2048, 16), (2500, 2, 24, 8, 1)]


def _index(rows, n, kind, gen):
    if kind == "idle":
        return torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    if kind == "last":
        return torch.full((rows,), n - 1, dtype=torch.int64, device="cuda")
    ids = torch.randint(-1, n, (rows,), generator=gen, device="cuda")
    return (torch.sort(ids)[0] if kind == "runs" else ids).to(torch.int32)


def _data(rows, n, k, m, r, dtype, kind="mixed", seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64).to(dtype)

    x, A, B, base, dy = rnd(rows, k), rnd(n, r, k), rnd(n, m, r), rnd(rows, m), rnd(rows, m)
    if dtype == torch.float16:
        A, dy = A / 16, dy / 16
    scale = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) + 0.5
    return x, A, B, base, dy, scale, _index(rows, n, kind, gen)


def _units(dtype):
    """(unit of a sum, half a step of the result, share lost by a split intermediate)"""
    e = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -23
    return e, torch.finfo(dtype).eps / 2, 2.0 ** -15 if dtype in (torch.float16, torch.bfloat16) else 0.0


def _close(got, want, magnitude, length, dtype, split=True):
    e, half, lost = _units(dtype)
    tol = half * want.abs() * (1 + 2 ** -6) + (e * (length + 8) * 2 + (lost if split else 0)) * magnitude \
        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    worst = ((got.double() - want).abs() - tol).max().item() if want.numel() else 0.0
    assert worst <= 0, f"off by {worst} more than allowed"


def _formula(x, A, B, base, scale, index):
    """y, its sums' magnitudes, u and |u| in float64, adapter by adapter."""
    xd, Ad, Bd = x.double(), A.double(), B.double()
    y = torch.zeros((x.shape[0], B.shape[1]), dtype=torch.float64, device="cuda") if base is None else base.double().clone()
    mag = y.abs()
    u = torch.zeros((x.shape[0], A.shape[1]), dtype=torch.float64, device="cuda")
    ua = torch.zeros_like(u)
    for i in range(A.shape[0]):
        t = index == i
        s = float(scale[i]) if isinstance(scale, torch.Tensor) else scale
        u[t] = s * xd[t] @ Ad[i].T
        ua[t] = abs(s) * xd[t].abs() @ Ad[i].abs().T
        y[t] += u[t] @ Bd[i].T
        mag[t] += ua[t] @ Bd[i].abs().T
    return y, mag, u, ua


@pytest.mark.parametrize("kind", ["mixed", "runs", "idle", "last"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(size, dtype, kind):
    rows, n, k, m, r = size
    x, A, B, base, _, scale, index = _data(rows, n, k, m, r, dtype, kind)
    want, mag, _, _ = _formula(x, A, B, base, scale, index)
    got = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    assert got.dtype == dtype and got.shape == base.shape
    _close(got, want, mag, k + r, dtype)
    idle = index == -1
    assert torch.equal(got[idle], base[idle])  # untouched, bit for bit
    again = fp.adapter_matmul(x, A, B, fp.prepare_rows(index, n), base=base, scale=scale)
    assert torch.equal(got, again)
    plain, pmag, _, _ = _formula(x, A, B, None, 0.5, index)
    _close(fp.adapter_matmul(x, A, B, index, scale=0.5), plain, pmag, k + r, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gradients_by_the_formula(size, dtype):
    rows, n, k, m, r = size
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, dtype, "mixed", 3)
    for t in (x, A, B, base):
        t.requires_grad_(True)
    y = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    dx, dA, dB, dbase = torch.autograd.grad(y, (x, A, B, base), dy)
    again = torch.autograd.grad(fp.adapter_matmul(x, A, B, index, base=base, scale=scale), (x, A, B), dy)
    assert all(torch.equal(a, b) for a, b in zip((dx, dA, dB), again))
    with torch.no_grad():
        want, mag, u, ua = _formula(x, A, B, base, scale, index)
        _close(y, want, mag, k + r, dtype)
        assert torch.equal(dbase, dy)
        # dx is the operator itself with the factors' roles exchanged
        dxw, dxm, v, va = _formula(dy, B.transpose(1, 2), A.transpose(1, 2), None, scale, index)
        _close(dx, dxw, dxm, m + r, dtype)
        for i in range(n):
            t = index == i
            _close(dA[i], v[t].T @ x[t].double(), va[t].T @ x[t].double().abs(), m + rows, dtype)
            _close(dB[i], dy[t].double().T @ u[t], dy[t].double().abs().T @ ua[t], k + rows, dtype)


def test_gradients_by_differences():
    x, A, B, base, _, scale, index = _data(300, 3, 5, 4, 2, torch.float64, "mixed", 5)
    x, A, B, base = (t.requires_grad_(True) for t in (x[:7], A, B, base[:7]))
    index = index[:7].clone()
    index[:3] = torch.arange(3, device="cuda")
    assert torch.autograd.gradcheck(lambda *a: fp.adapter_matmul(*a[:3], index, base=a[3], scale=scale), (x, A, B, base))


@pytest.mark.parametrize("rows", [9, 400])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides_alignment_and_in_place(dtype, rows):
    n, k, m, r = 3, 70, 50, 5
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, dtype, "mixed", 7)
    want = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)

    def odd(t):  # the same values one element past an aligned start, with a gap after each row
        wide = torch.zeros(t.shape[:-1] + (t.shape[-1] + 3,), dtype=dtype, device="cuda").flatten()
        wide = torch.cat([wide, wide[:1]])[1:].view(t.shape[:-1] + (t.shape[-1] + 3,))
        view = wide[..., :t.shape[-1]]
        view.copy_(t)
        return view

    want_mag = _formula(x, A, B, base, scale, index)[1]
    for a, b, c, d in ((odd(x), A, B, base), (x, odd(A), odd(B), base), (x, A, B, odd(base)),
                       (x.T.contiguous().T, A.transpose(1, 2).contiguous().transpose(1, 2), odd(B), odd(base))):
        got = fp.adapter_matmul(a, b, c, index, base=d, scale=scale)
        _close(got, want.double(), want_mag, k + r, dtype)
    out = odd(torch.zeros_like(base))
    gap = out.as_strided((rows, 3), (out.stride(0), 1), out.storage_offset() + m)[:-1].clone()
    assert fp.adapter_matmul(x, A, B, index, base=base, scale=scale, out=out) is out
    _close(out, want.double(), want_mag, k + r, dtype)
    assert torch.equal(out.as_strided((rows, 3), (out.stride(0), 1), out.storage_offset() + m)[:-1], gap)
    in_place = base.clone()
    version = in_place._version
    fp.adapter_matmul(x, A, B, index, base=in_place, scale=scale, out=in_place)
    assert torch.equal(in_place, want) and in_place._version > version
    # one row for all: a stride of zero
    same = fp.adapter_matmul(x[:1].expand(rows, k), A, B, index, base=base[0], scale=scale)
    w, mag, _, _ = _formula(x[:1].expand(rows, k), A, B, base[0].expand(rows, m), scale, index)
    _close(same, w, mag, k + r, dtype)
    with pytest.raises(RuntimeError, match="overlaps"):
        fp.adapter_matmul(x, A, B, index, base=base, out=x[:, :m] if k == m else x.flatten()[:rows * m].view(rows, m))


def test_leading_shapes_and_broadcast_gradients():
    b, s, n, k, m, r = 3, 100, 4, 32, 24, 4
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(b, s, k, generator=gen, device="cuda", dtype=torch.float64, requires_grad=True)
    A = torch.randn(n, r, k, generator=gen, device="cuda", dtype=torch.float64, requires_grad=True)
    B = torch.randn(n, m, r, generator=gen, device="cuda", dtype=torch.float64, requires_grad=True)
    bias = torch.randn(m, generator=gen, device="cuda", dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([2, -1, 2], device="cuda")
    y = fp.adapter_matmul(x, A, B, ids, base=bias)
    y2 = fp.adapter_matmul(x, A, B, fp.prepare_rows(ids, n, (b, s)), base=bias)
    assert y.shape == (b, s, m) and torch.equal(y, y2)
    want, mag, _, _ = _formula(x.detach().view(-1, k), A.detach(), B.detach(), bias.detach().expand(b * s, m), 1.0,
                               ids.repeat_interleave(s))
    _close(y.detach().view(-1, m), want, mag, k + r, torch.float64)
    g = torch.autograd.grad(y.sum(), (x, A, B, bias))  # an expanded gradient of ones
    assert torch.equal(g[3], torch.full_like(bias, b * s))
    assert torch.count_nonzero(g[1][[0, 1, 3]]) == 0 and torch.count_nonzero(g[2][[0, 1, 3]]) == 0
    only_b = torch.autograd.grad(fp.adapter_matmul(x.detach(), A.detach(), B, ids, base=bias.detach()).sum(), B)[0]
    assert torch.equal(only_b, g[2])
    only_a = torch.autograd.grad(fp.adapter_matmul(x.detach(), A, B.detach(), ids).sum(), A)[0]
    assert torch.equal(only_a, g[1])
    one = fp.adapter_matmul(x.detach()[0, 0], A.detach(), B.detach(), torch.tensor(2, device="cuda"), base=bias.detach())
    _close(one, want[0], mag[0], k + r, torch.float64)
    empty = fp.adapter_matmul(x.detach()[:0], A.detach(), B.detach(), ids[:0], base=bias.detach())
    assert empty.shape == (0, s, m)
    zero_k = fp.adapter_matmul(x.detach()[..., :0], A.detach()[..., :0], B.detach(), ids, base=bias.detach())
    assert torch.equal(zero_k, bias.detach().expand(b, s, m))
    assert fp.adapter_matmul(x.detach(), A.detach(), B.detach()[:, :0], ids).shape == (b, s, 0)


def test_no_rows_give_zero_gradients():
    A = torch.ones(2, 3, 8, device="cuda", dtype=torch.float64, requires_grad=True)
    B = torch.ones(2, 5, 3, device="cuda", dtype=torch.float64, requires_grad=True)
    x = torch.ones(0, 8, device="cuda", dtype=torch.float64)
    y = fp.adapter_matmul(x, A, B, torch.zeros(0, dtype=torch.int32, device="cuda"))
    dA, dB = torch.autograd.grad(y.sum(), (A, B))
    assert torch.count_nonzero(dA) == 0 and torch.count_nonzero(dB) == 0 and dA.shape == A.shape


@pytest.mark.parametrize("rows", [33, 500])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_what_other_rows_hold_stays_out(dtype, rows):
    """NaN and infinities in one row, one adapter or the padding reach only their own rows."""
    n, k, m, r = 4, 96, 40, 6
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, dtype, "mixed", 9)
    index[:8] = torch.tensor([0, 1, 2, 3, -1, 0, 1, -1], device="cuda")
    want = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    x2, A2, B2 = x.clone(), A.clone(), B.clone()
    x2[0] = float("nan")
    x2[4] = float("inf")
    A2[3] = float("nan")
    B2[2, 0] = float("inf")
    got = fp.adapter_matmul(x2, A2, B2, index, base=base, scale=scale)
    clean = (index != 3) & (index != 2)
    clean[0] = False
    assert torch.equal(got[clean], want[clean])
    assert torch.isnan(got[0]).all() and torch.isnan(got[index == 3]).all()
    rest = index == 2
    assert torch.equal(got[rest][:, 1:], want[rest][:, 1:]) and not torch.isfinite(got[rest][:, 0]).any()
    # a row's own infinity stays one where every product is of its sign
    one = torch.full((1, 1), float("inf"), dtype=dtype, device="cuda")
    got = fp.adapter_matmul(one.expand(rows, 1), A.abs()[..., :1] + 1, B.abs() + 1, index, base=base, scale=scale)
    assert torch.isposinf(got[index >= 0]).all() and torch.equal(got[index < 0], base[index < 0])
    for t in (x2, A2, B2):
        t.requires_grad_(True)
    dx, dA, dB = torch.autograd.grad(fp.adapter_matmul(x2, A2, B2, index, base=base, scale=scale), (x2, A2, B2), dy)
    assert torch.isfinite(dA[1]).all() and torch.isfinite(dB[1]).all() and torch.isnan(dA[0]).any()
    assert torch.equal(dx[4], torch.zeros_like(dx[4]))


@pytest.mark.parametrize("rows", [20, 400])
def test_bad_ids_become_nan_and_an_error(rows, monkeypatch):
    from fp_emulation import ozaki

    n, k, m, r = 3, 16, 16, 4
    x, A, B, base, _, scale, index = _data(rows, n, k, m, r, torch.float64, "mixed", 11)
    want = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
    bad = index.to(torch.int64)
    wrong = torch.tensor([3, 7, 11], device="cuda")
    bad[wrong] = torch.tensor([n, -2, (1 << 32) + 1], device="cuda")
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[wrong] = False
    for prepared in (False, True):
        monkeypatch.setattr(ozaki, "_CHECK_MODE", "off")
        got = fp.adapter_matmul(x, A, B, fp.prepare_rows(bad, n) if prepared else bad, base=base, scale=scale)
        assert torch.isnan(got[wrong]).all() and torch.equal(got[keep], want[keep])
        monkeypatch.setattr(ozaki, "_CHECK_MODE", "poll")
        with pytest.raises(_lib.FpemuError, match="adapter id"):
            fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        assert _lib.device_error(clear=True)[0] == 0  # raised once, and cleared
        assert torch.equal(fp.adapter_matmul(x, A, B, index, base=base, scale=scale), want)


@pytest.mark.parametrize("rows", [32, 600])
def test_captured_and_replayed(rows):
    n, k, m, r = 5, 128, 96, 8
    x, A, B, base, dy, scale, index = _data(rows, n, k, m, r, torch.bfloat16, "mixed", 13)
    prepared = fp.prepare_rows(index, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fp.adapter_matmul(x, A, B, index, base=base, scale=scale)
        fp.adapter_matmul(x, A, B, prepared, base=base, scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = fp.adapter_matmul(x, A, B, index, base=base, scale=scale)  # groups the rows at every replay
    with torch.cuda.graph(g2):
        y2 = fp.adapter_matmul(x, A, B, prepared, base=base, scale=scale)
    for seed in (14, 15):
        new = _data(rows, n, k, m, r, torch.bfloat16, "mixed", seed)
        x.copy_(new[0])
        base.copy_(new[3])
        g2.replay()
        assert torch.equal(y2, fp.adapter_matmul(x, A, B, prepared, base=base, scale=scale))
        index.copy_(new[6])
        g1.replay()
        g1.replay()
        assert torch.equal(y1, fp.adapter_matmul(x, A, B, index, base=base, scale=scale))


def test_two_streams_at_once():
    sets = [_data(rows, 4, 256, 512, 16, torch.float64, "mixed", rows) for rows in (200, 3000)]
    want = [fp.adapter_matmul(s[0], s[1], s[2], s[6], base=s[3], scale=s[5]) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(fp.adapter_matmul(s[0], s[1], s[2], s[6], base=s[3], scale=s[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


def test_refusals():
    x, A, B, base, _, scale, index = _data(6, 3, 8, 5, 2, torch.float64)
    ok = dict(base=base, scale=scale)
    with pytest.raises(TypeError):
        fp.adapter_matmul(x, A.float(), B, index, **ok)
    with pytest.raises(TypeError):
        fp.adapter_matmul(x, A, B, index.float(), **ok)
    with pytest.raises(TypeError):
        fp.adapter_matmul(x, A, B, [0] * 6, **ok)
    with pytest.raises(RuntimeError):
        fp.adapter_matmul(x, A, B[:2], index, **ok)
    with pytest.raises(RuntimeError):
        fp.adapter_matmul(x[:, :7], A, B, index, **ok)
    with pytest.raises(RuntimeError):
        fp.adapter_matmul(x, A, B, index[:5], **ok)
    with pytest.raises(RuntimeError):
        fp.adapter_matmul(x, A, B, index, base=base, scale=scale[:2])
    with pytest.raises(RuntimeError):
        fp.adapter_matmul(x, A, B, fp.prepare_rows(index, 4), **ok)
    with pytest.raises(RuntimeError):
        fp.adapter_matmul(x, A, B, fp.prepare_rows(index[:4], 3), **ok)
    with pytest.raises(RuntimeError, match="different devices|CUDA"):
        fp.adapter_matmul(x, A, B.cpu(), index, **ok)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp.adapter_matmul(x, A, B, index.cpu(), **ok)
    with pytest.raises(RuntimeError, match="gradient"):
        fp.adapter_matmul(x, A, B, index, base=base, scale=scale.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="out"):
        fp.adapter_matmul(x, A.clone().requires_grad_(True), B, index, base=base, out=base.clone())
    with pytest.raises(ValueError):
        fp.adapter_matmul(x, A[:, :0], B[..., :0], index, **ok)
    big = torch.zeros(3, 129, 8, dtype=torch.float64, device="cuda")
    with pytest.raises(ValueError):
        fp.adapter_matmul(x, big, torch.zeros(3, 5, 129, dtype=torch.float64, device="cuda"), index, **ok)
    x.requires_grad_(True)
    g, = torch.autograd.grad(fp.adapter_matmul(x, A, B, index, **ok).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def _model(seed=0):
    torch.manual_seed(seed)
    layers = torch.nn.Sequential(torch.nn.Linear(2, 64, dtype=torch.float64), torch.nn.Tanh(),
                                 torch.nn.Linear(64, 48, dtype=torch.float64), torch.nn.Tanh(),
                                 torch.nn.Linear(48, 1, dtype=torch.float64)).cuda()
    return fp.convert(layers)


def test_linear_layers_with_adapters():
    model = _model()
    x = torch.randn(3, 40, 2, device="cuda", dtype=torch.float64)
    plain = model(x).detach()
    fp.add_adapters(model, 4, rank=3, alpha=6)
    ids = torch.tensor([1, -1, 3], device="cuda")
    assert torch.equal(model(x), plain)
    with fp.use_adapters(model, ids):
        assert torch.equal(model(x), plain)  # B starts at zero
    for layer in model:
        if isinstance(layer, fp.Linear):
            torch.nn.init.normal_(layer.adapters.B, std=0.3)

    def by_hand(h):
        for layer in model:
            if isinstance(layer, fp.Linear):
                add = torch.zeros(h.shape[:-1] + (layer.out_features,), dtype=torch.float64, device="cuda")
                for i, a in enumerate(ids.tolist()):
                    if a >= 0:
                        add[i] = 2.0 * (h[i] @ layer.adapters.A[a].T) @ layer.adapters.B[a].T
                h = h @ layer.weight.T + layer.bias + add
            else:
                h = layer(h)
        return h

    want = by_hand(x).detach()
    with fp.use_adapters(model, ids), torch.no_grad():
        frozen = model(x)
    with fp.use_adapters(model, ids):
        recorded = model(x)
    assert torch.equal(frozen, recorded)
    # three layers of at most 64 + 3 products of magnitude below 10: 2^-53 * 70 * 10, carried through them
    assert (recorded - want).abs().max() < 1e-12 and torch.equal(recorded[1], plain[1])
    assert not torch.equal(recorded[0], plain[0]) and torch.equal(model(x), plain)
    names = [k for k in model.state_dict() if "adapters" in k]
    assert names == [f"{i}.adapters.{f}" for i in (0, 2, 4) for f in "AB"]


def test_fine_tuning_steps_together():
    """Adapters trained beside frozen layers, the gradients clipped, against the same steps in plain float64."""
    model = _model(3)
    model.requires_grad_(False)
    fp.add_adapters(model, 3, rank=2)
    for layer in model:
        if isinstance(layer, fp.Linear):
            torch.nn.init.normal_(layer.adapters.B, std=0.5)
    import copy

    twin = copy.deepcopy(model)
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(400, 2, generator=gen, device="cuda", dtype=torch.float64)
    ids = torch.randint(-1, 3, (400,), generator=gen, device="cuda")
    target = torch.randn(400, 1, generator=gen, device="cuda", dtype=torch.float64)
    params = [p for p in model.parameters() if p.requires_grad]
    mirror = [p for p in twin.parameters() if p.requires_grad]
    assert len(params) == 6
    opt, opt2 = torch.optim.SGD(params, lr=0.1), torch.optim.SGD(mirror, lr=0.1)
    for _ in range(3):
        opt.zero_grad()
        with fp.use_adapters(model, ids):
            loss = ((model(x) - target) ** 2).sum()
        loss.backward()
        norm = fp.clip_grad_norm_(params, 1.0)
        opt.step()

        opt2.zero_grad()
        h = x
        for layer in twin:
            if isinstance(layer, fp.Linear):
                y = h @ layer.weight.T + layer.bias
                A, B = layer.adapters.A, layer.adapters.B
                one_hot = torch.nn.functional.one_hot(ids.clamp(min=0), 3).double() * (ids >= 0).double()[:, None]
                h = y + torch.einsum("tk,ark,aor,ta->to", h, A, B, one_hot)
            else:
                h = layer(h)
        ((h - target) ** 2).sum().backward()
        norm2 = torch.nn.utils.clip_grad_norm_(mirror, 1.0)
        opt2.step()
        assert norm > 1 and torch.isclose(norm, norm2, rtol=1e-10, atol=0)
        for p, q in zip(params, mirror):
            assert torch.allclose(p.grad, q.grad, rtol=1e-9, atol=1e-12)
            assert torch.allclose(p, q, rtol=1e-9, atol=1e-12)
