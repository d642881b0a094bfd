"""What the adapter products keep of the rank-long intermediate u = s A x, shown
where its leading bits cancel.

Every number below is a sum of few powers of two, chosen so that each product and
each partial sum is exact in 24 bits: an evaluation that holds u as a float gives
the expected value itself, with no rounding anywhere."""
from __future__ import annotations

import pytest
import torch

import fp_emulation as fp

pytestmark = pytest.mark.gpu

ROWS = [1, 9, 200, 257, 3000]


def _cancelling(rows, p, k, m):
    """u = (1 + 2^-8 + 2^-p, -(1 + 2^-8)); with B = (1, 1) only 2^-p is left."""
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[:, :3] = 1
    A = torch.zeros(1, 2, k, dtype=torch.bfloat16, device="cuda")
    A[0, 0, :3] = torch.tensor([1.0, 2.0 ** -8, 2.0 ** -p])
    A[0, 1, :2] = torch.tensor([-1.0, -(2.0 ** -8)])
    B = torch.ones(1, m, 2, dtype=torch.bfloat16, device="cuda")
    return x, A, B, torch.zeros(rows, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("p", [12, 16, 18, 20])
@pytest.mark.parametrize("rows", ROWS)
def test_bfloat16_middle_has_the_bits_of_a_float(rows, p):
    x, A, B, index = _cancelling(rows, p, 40, 24)
    y = fp.adapter_matmul(x, A, B, index)
    assert torch.equal(y, torch.full_like(y, 2.0 ** -p))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows", ROWS)
def test_infinite_bfloat16_row_keeps_its_sign(rows, sign):
    """Weights of 8: no part of the infinite u may overflow to the other sign."""
    x = torch.full((rows, 1), sign * float("inf"), dtype=torch.bfloat16, device="cuda")
    A = torch.ones(1, 1, 1, dtype=torch.bfloat16, device="cuda")
    B = torch.full((1, 20, 1), 8.0, dtype=torch.bfloat16, device="cuda")
    y = fp.adapter_matmul(x, A, B, torch.zeros(rows, dtype=torch.int32, device="cuda"))
    assert torch.equal(y, torch.full_like(y, sign * float("inf")))


@pytest.mark.parametrize("p", [16, 20])
@pytest.mark.parametrize("rows", [2, 64, 512, 2048])
def test_bfloat16_gradients_have_the_bits_of_a_float(rows, p):
    """Rows in pairs whose u, and whose v = B^T dy, are 1 + 2^-8 + 2^-p and -(1 + 2^-8); the
    gradients' sums over a pair are 2^-p.  dx is the product of test_bfloat16_middle."""
    power = torch.tensor([1.0, 2.0 ** -8, 2.0 ** -p], dtype=torch.bfloat16, device="cuda")
    pair = torch.stack([power, torch.cat([-power[:2], power.new_zeros(1)])])
    x = pair.repeat(rows // 2, 1)
    dy = x.clone()
    A = torch.ones(1, 1, 3, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    B = torch.ones(1, 3, 1, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    index = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ones = torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda")
    want = rows // 2 * 2.0 ** -p
    dB, = torch.autograd.grad(fp.adapter_matmul(x, A, B[:, :1], index), B, ones)
    assert torch.equal(dB[:, :1], torch.full_like(dB[:, :1], want))
    dA, = torch.autograd.grad(fp.adapter_matmul(ones, A[..., :1], B, index), A, dy)
    assert torch.equal(dA[..., :1], torch.full_like(dA[..., :1], want))
    A2 = torch.ones(1, 2, 1, dtype=torch.bfloat16, device="cuda")
    B2 = torch.stack([torch.ones(3), torch.tensor([-1.0, -1.0, 0.0])], 1)[None].to(A2)
    ones.requires_grad_(True)
    dx, = torch.autograd.grad(fp.adapter_matmul(ones, A2, B2, index), ones, power.expand(rows, 3))
    assert torch.equal(dx, torch.full_like(dx, 2.0 ** -p))


@pytest.mark.parametrize("long", [False, True], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_long_sums_of_one_sign(dtype, long):
    """u_0 adds 65536 positive products, u_1 subtracts their exact sum S in up to four pieces, and y is
    what u_0 is off by.  Tolerance: the tensor cores' adders keep 22 bits or more, and a block joins
    their sums after 64 of their instructions at most (24 for floats), into a float that is rounded
    to nearest (at most 128 times); a float's product is off by 2^-21 of it."""
    k, m = 65536, 8
    n, rows = (1, 64 * 300) if long else (200, 200)  # whole sums in one block
    gen = torch.Generator(device="cuda").manual_seed(1)

    def ones(*shape):
        return (torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64) + 1).to(dtype)

    x = ones(1, k)
    x[:, :4] = 1
    A = torch.zeros(n, 2, k, dtype=dtype, device="cuda")
    A[:, 0] = ones(n, k) * 2.0 ** -6
    rest = (x.double() * A[:, 0].double()).sum(1)
    total = rest.clone()
    for j in range(4):
        A[:, 1, j] = -rest.to(dtype)
        rest = rest + A[:, 1, j].double()
    assert (rest.abs() <= 2.0 ** -23 * total).all()
    index = torch.arange(rows, dtype=torch.int32, device="cuda") % n
    y = fp.adapter_matmul(x.expand(rows, k), A, torch.ones(n, m, 2, dtype=dtype, device="cuda"), index)
    off = (y.double() / total[index.long()][:, None]).abs().max().item()
    adds = 24 if dtype == torch.float32 else 64
    assert off <= adds * 2.0 ** -22 + 128 * 2.0 ** -24 + 2.0 ** -21


@pytest.mark.parametrize("apart", [4, 12, 16, 18, 24, 28])
@pytest.mark.parametrize("rows", ROWS)
def test_half_middle_of_far_magnitudes(rows, apart):
    """u = (2^a, 2^-b (1 + 2^-9)), b + a = apart; B takes the second alone, which a half holds."""
    b = min(apart, 14)
    x = torch.tensor([1.0, 1 + 2.0 ** -9], dtype=torch.float16, device="cuda").expand(rows, 2)
    A = torch.tensor([[[2.0 ** (apart - b), 0], [0, 2.0 ** -b]]], dtype=torch.float16, device="cuda")
    B = torch.tensor([0, 2.0 ** 10], dtype=torch.float16, device="cuda").expand(1, 20, 2)
    y = fp.adapter_matmul(x, A, B, torch.zeros(rows, dtype=torch.int32, device="cuda"))
    assert torch.equal(y, torch.full_like(y, 2.0 ** (10 - b) * (1 + 2.0 ** -9)))


@pytest.mark.parametrize("rows", ROWS)
def test_half_middle_beside_an_infinity(rows):
    """u = (inf, 3.6e9): the second is finite, and takes nothing from the first."""
    x = torch.tensor([1.0, 60000.0], dtype=torch.float16, device="cuda").expand(rows, 2)
    A = torch.tensor([[[float("inf"), 0], [0, 60000.0]]], dtype=torch.float16, device="cuda")
    B = torch.tensor([1.0, -1.0], dtype=torch.float16, device="cuda").expand(1, 20, 2)
    y = fp.adapter_matmul(x, A, B, torch.zeros(rows, dtype=torch.int32, device="cuda"))
    assert torch.equal(y, torch.full_like(y, float("inf")))
