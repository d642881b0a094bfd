"""The global gradient norm and clipping on the GPU, against exact sums.

Tolerances: every element enters a double; a thread adds at most 64 of them per
chunk before the sums are joined pairwise, so the sum of n positive terms below
2^20 in all is off by at most 128 * 2^-53 of itself, the norm by that or less.  A
scaled element is off by the factor's error and one rounding of its type."""
from __future__ import annotations

import math

import pytest
import torch

import fp_emulation as fp

pytestmark = pytest.mark.gpu

ALL = [torch.float64, torch.float32, torch.float16, torch.bfloat16]
NORM_TOL = 128 * 2.0 ** -53


def _exact(tensors, p):
    values = torch.cat([t.detach().double().abs().flatten().cpu() for t in tensors]).tolist()
    if p == math.inf:
        return max(values, default=0.0)
    if p == 1:
        return math.fsum(values)
    top = max(values, default=0.0)
    if top == 0 or not math.isfinite(top):
        return top
    e = math.frexp(top)[1]
    return math.ldexp(math.sqrt(math.fsum(math.ldexp(v, -e) ** 2 for v in values)), e)


def _tensors(sizes, dtypes, seed=0, std=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=gen, device="cuda", dtype=torch.float64) * std).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def _check_scaled(got, src, c):
    for o, g in zip(got, src):
        want = g.double() * c
        half = torch.finfo(g.dtype).eps / 2
        extra = 2 * NORM_TOL if g.dtype == torch.float64 else 2.0 ** -40 if g.dtype == torch.float32 else 2.0 ** -23
        tol = (half + extra) * want.abs() + torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps
        assert o.dtype == g.dtype and ((o.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("p", [1, 2, math.inf])
@pytest.mark.parametrize("dtypes", [[d] for d in ALL] + [ALL], ids=str)
def test_norm_and_scaling(dtypes, p):
    sizes = [1, 0, 7, 8, 9, 255, 256, 257, 16383, 16384, 16385, 70001, 3, 0, 5]
    grads = _tensors(sizes, dtypes)
    want = _exact(grads, p)
    norm = fp.grad_norm(grads, p)
    wide = torch.float64 if torch.float64 in dtypes else torch.float32
    assert norm.dtype == wide and norm.shape == () and norm.is_cuda
    tol = NORM_TOL if wide == torch.float64 else 2.0 ** -24 + NORM_TOL
    assert abs(norm.item() - want) <= tol * want
    keep = [g.clone() for g in grads]
    for share in (0.37, 1.0, 2.0):
        limit = want * share
        c = min(1.0, limit / (want + 1e-6))
        out, n2 = fp.clip_grads(grads, limit, p)
        assert torch.equal(n2, norm) and all(torch.equal(a, b) for a, b in zip(grads, keep))
        _check_scaled(out, grads, c)
        params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
        for q, g in zip(params, grads):
            q.grad = g.clone()
        versions = [q.grad._version for q in params]
        assert torch.equal(fp.clip_grad_norm_(params, limit, p), norm)
        assert all(torch.equal(q.grad, o) for q, o in zip(params, out))
        assert all(q.grad._version > v for q, v in zip(params, versions))
    assert all(torch.equal(a, b) for a, b in zip(fp.clip_grads(grads, want * 2, p)[0], keep))


def test_agrees_with_torch():
    params = [torch.nn.Parameter(torch.empty(n, device="cuda")) for n in (1000, 3, 77777)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda")
    twins = [torch.nn.Parameter(torch.empty_like(p)) for p in params]
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    a, b = fp.clip_grad_norm_(params, 2.5), torch.nn.utils.clip_grad_norm_(twins, 2.5)
    assert a.dtype == b.dtype and torch.isclose(a, b, rtol=1e-5, atol=0)
    assert all(torch.allclose(p.grad, q.grad, rtol=1e-5, atol=0) for p, q in zip(params, twins))


def test_many_tensors_in_several_launches():
    grads = _tensors([(i * 37) % 300 for i in range(1200)], ALL, 2)
    want = _exact(grads, 2)
    out, norm = fp.clip_grads(grads, 1.0)
    assert abs(norm.item() - want) <= NORM_TOL * want
    _check_scaled(out, grads, 1.0 / (want + 1e-6))
    assert torch.equal(fp.grad_norm(grads), norm)


@pytest.mark.parametrize("shift", [0, 1, 3, 5])
@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_packed_views_of_any_alignment(dtype, shift):
    flat = _tensors([50000], [dtype], 3)[0]
    views, at = [], shift
    for n in (1, 2, 16385, 7, 20000):
        views.append(flat[at:at + n])
        at += n
    before, rest = flat.clone(), torch.ones(50000, dtype=torch.bool, device="cuda")
    rest[shift:at] = False
    want = _exact(views, 2)
    out, norm = fp.clip_grads(views, want / 3)
    assert abs(norm.item() - want) <= (NORM_TOL if dtype == torch.float64 else 2.0 ** -24 + NORM_TOL) * want
    _check_scaled(out, views, want / 3 / (want + 1e-6))
    away = torch.empty(60000, dtype=dtype, device="cuda")[shift // 2 + 1:]
    places = [away[sum(v.numel() for v in views[:i]):][:v.numel()] for i, v in enumerate(views)]
    assert all(torch.equal(a, b) for a, b in zip(fp.clip_grads(views, want / 3, out=places)[0], out))
    assert torch.equal(flat, before)
    same, _ = fp.clip_grads(views, want / 3, out=views)
    assert all(torch.equal(a, b) for a, b in zip(same, out)) and torch.equal(flat[rest], before[rest])


def test_memory_orders_and_gaps():
    gen = torch.Generator(device="cuda").manual_seed(4)
    whole = torch.randn(6, 8, 10, 12, generator=gen, device="cuda")
    grads = [whole[:2].clone().to(memory_format=torch.channels_last), whole[2:4, ::2], whole[4].transpose(0, 2),
             torch.ones(1, device="cuda").expand(50)]
    want = _exact(grads, 2)
    out, norm = fp.clip_grads(grads, 1.0)
    assert abs(norm.item() - want) <= (2.0 ** -24 + NORM_TOL) * want
    _check_scaled(out, grads, 1 / (want + 1e-6))
    kept = whole.clone()
    values = [g.clone() for g in grads[:3]]
    c = 1 / (_exact(values, 2) + 1e-6)
    fp.clip_grads(grads[:3], 1.0, out=grads[:3])
    _check_scaled(grads[:3], values, c)
    assert torch.equal(whole[:2], kept[:2]) and torch.equal(whole[5], kept[5]) and torch.equal(whole[2:4, 1::2], kept[2:4, 1::2])


@pytest.mark.parametrize("exponent", [-320, -300, -150, 0, 150, 290, 307])
def test_far_magnitudes_of_doubles(exponent):
    base = torch.rand(3000, dtype=torch.float64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) / 64
    g = base * 10.0 ** exponent
    want = _exact([g], 2)
    got = fp.grad_norm([g]).item()
    # below the normal range the elements and the result are whole steps of 2^-1074
    assert abs(got - want) <= NORM_TOL * want + 2.0 ** -1074
    if exponent in (150, 290):
        out, _ = fp.clip_grads([g], 1.0)
        _check_scaled(out, [g], 1.0 / (want + 1e-6))
    mixed = torch.cat([g, base])
    want = _exact([mixed], 2)
    assert abs(fp.grad_norm([mixed]).item() - want) <= NORM_TOL * want


def test_range_of_narrow_types():
    big = torch.full((4,), 3e38, device="cuda")
    assert fp.grad_norm([big]).item() == math.inf  # 6e38 is no float
    assert abs(fp.grad_norm([big, torch.zeros(1, dtype=torch.float64, device="cuda")]).item() / (2 * big[0].item()) - 1) < 1e-15
    tiny = torch.full((100,), 2.0 ** -133, dtype=torch.bfloat16, device="cuda")
    assert fp.grad_norm([tiny]).item() == 10 * 2.0 ** -133
    assert fp.grad_norm([torch.full((10000,), 65504.0, dtype=torch.float16, device="cuda")]).item() == 6550400.0
    assert fp.grad_norm([torch.zeros(10, device="cuda")]).item() == 0


@pytest.mark.parametrize("p", [1, 2, math.inf])
@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_non_finite(dtype, p):
    for value, clipped in ((math.nan, math.nan), (math.inf, 0.0), (-math.inf, 0.0)):
        grads = _tensors([100, 20000], [dtype], 6)
        grads[1][17000] = value
        out, norm = fp.clip_grads(grads, 1.0, p)
        assert (math.isnan(norm.item()) if math.isnan(value) else norm.item() == math.inf)
        if math.isnan(value):
            assert torch.isnan(out[0]).all() and torch.isnan(out[1]).all()
        else:  # c = 0, as torch.nn.utils: zeros, and NaN in the infinity's place
            assert torch.count_nonzero(out[0]) == 0 and torch.isnan(out[1][17000])
        q = torch.nn.Parameter(torch.empty_like(grads[1]))
        q.grad = grads[1].clone()
        with pytest.raises(RuntimeError, match="non-finite"):
            fp.clip_grad_norm_([q], 1.0, p, error_if_nonfinite=True)
        assert torch.equal(q.grad.nan_to_num(), grads[1].nan_to_num())


def test_in_bounds_gradients_stay_and_limits():
    grads = _tensors([5000, 3], [torch.float64, torch.bfloat16], 7)
    keep = [g.clone() for g in grads]
    fp.clip_grads(grads, math.inf, out=grads)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    out, _ = fp.clip_grads(grads, 0.0)
    assert all(torch.count_nonzero(o) == 0 for o in out)


def test_repeats_and_replays():
    grads = _tensors([100001, 33, 40000], ALL, 8)
    out, norm = fp.clip_grads(grads, 1.0)
    for _ in range(3):
        out2, norm2 = fp.clip_grads(grads, 1.0)
        assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(out, out2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, held_norm = fp.clip_grads(grads, 1.0)
    for g, new in zip(grads, _tensors([100001, 33, 40000], ALL, 9)):
        g.copy_(new)
    graph.replay()
    out, norm = fp.clip_grads(grads, 1.0)
    assert torch.equal(norm, held_norm) and all(torch.equal(a, b) for a, b in zip(out, held))
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                results.append(fp.clip_grads(grads, 1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(o, out)) for o, n in results)


def test_refusals():
    g = torch.ones(10, device="cuda")
    p = torch.nn.Parameter(torch.empty(10, device="cuda"))
    p.grad = g
    with pytest.raises(ValueError, match="overlaps"):
        fp.clip_grad_norm_([p, p], 1.0)
    with pytest.raises(ValueError, match="overlaps"):
        fp.clip_grads([g[:5], g[5:]], 1.0, out=[g[5:], g[:5]])
    with pytest.raises(RuntimeError):
        fp.clip_grads([g], 1.0, out=[g, g])
    with pytest.raises(RuntimeError):
        fp.clip_grads([g], 1.0, out=[torch.ones(9, device="cuda")])
    with pytest.raises(RuntimeError):
        fp.clip_grads([g], 1.0, out=[torch.ones(10, device="cuda", dtype=torch.float64)])
    with pytest.raises(RuntimeError, match="CUDA"):
        fp.grad_norm([g, g.cpu()])
    with pytest.raises(TypeError):
        fp.grad_norm([g.to_sparse()])
    with pytest.raises(TypeError):
        fp.grad_norm([g.to(torch.complex64)])
    assert torch.equal(g, torch.ones(10, device="cuda"))
    assert fp.grad_norm([g, g]).item() == pytest.approx(math.sqrt(20), rel=1e-6)  # a norm alone may repeat one
