"""One rounding of the adapters' results: u = s x A^T (and v = s dy B) enters the products with 16 bits, not rounded to bf16.

Tolerance per output element, h = eps / 2 of the type: h |y| (its rounding) + h^2 sum_r |u_r| |B_r| (u = hi + lo, hi cut off towards zero, so lo is below
a step, 2 h |u|, and its own rounding below half a step of that: h^2 |u|) + n 2^-23 S (float32 accumulation of n terms of total size S); 2 % for
products of these errors.  In float32 u is one number: the same bound holds with its rounding, 2^-24 of sum |u| |B|, inside n 2^-23 S."""
import pytest
import torch

from test_adapters_gpu import BF, DEV, F32, ops, problem

pytestmark = pytest.mark.gpu


def oracle2(x, w, bias, a, b, scale, row):
    """(y, bound) in float64, on the tensors' device"""
    h = torch.finfo(x.dtype).eps / 2
    K, R = x.shape[1], a.shape[1]
    xd, wd = x.double(), w.double()
    y, S = xd @ wd.t(), xd.abs() @ wd.abs().t()
    U = torch.zeros_like(y)
    if bias is not None:
        y, S = y + bias.double(), S + bias.double().abs()
    for i in range(a.shape[0]):
        m = row == i
        ad, bd = a[i].double(), b[i].double()
        u = scale[i] * (xd[m] @ ad.t())
        y[m] += u @ bd.t()
        U[m] = u.abs() @ bd.abs().t()
        S[m] += abs(scale[i]) * (xd[m].abs() @ ad.abs().t()) @ bd.abs().t()
    return y, 1.02 * h * (y.abs() + h * U) + (2 * R + K + 4) * 2.0 ** -23 * S


def check(got, want, tol):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


CASES = [
    # lengths, ids, K, N, r, dtype
    ([1, 1], [1, 0], 1536, 516, 16, BF),
    ([1] * 8, [3, 0, -1, 4, 1, 0, 2, 5], 520, 772, 32, BF),
    ([7, 9], [1, 0], 4096, 96, 100, BF),
    ([3, 0, 61], [0, 1, 1], 128, 128, 8, BF),
    ([129, 0, 77, 300], [0, 0, -1, 1], 200, 132, 20, BF),
    ([300, 1, 212, 190], [1, 0, -1, 2], 192, 776, 48, BF),
    ([986], [0], 1024, 1540, 112, BF),
    ([1] * 600, [i % 5 - 1 for i in range(600)], 128, 520, 80, BF),
    ([4100], [0], 1984, 2052, 16, BF),                                  # the 256 x 256 tiles: ranks behind the K loop,
    ([4100], [0], 1984, 2052, 32, BF),                                  # ... in it,
    ([4100], [0], 2048, 2052, 144, BF),                                 # ... in both,
    ([1000, 1, 2000, 0, 1099], [1, 0, -1, 2, 1], 1984, 2052, 72, BF),   # ... tiles of several adapters
    ([3838, 1, 6, 5], [0, 1, -1, 2], 1024, 4100, 64, BF),               # ... and the rows behind whole rounds of them
    ([9, 4], [0, 1], 516, 36, 5, F32),
    ([300, 290], [0, 1], 100, 260, 40, F32),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_backward_round_once(case):
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids, K, N, r, dt = CASES[case]
    x, w, bias, a, b, scale, row = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in problem(lengths, ids, K, N, r, dt))
    dy = torch.randn(x.shape[0], N, generator=torch.Generator().manual_seed(9)).to(dt).to(DEV)
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale)
    y = o.linear_adapters(x, w, bias, bank, plan)
    check(y, *oracle2(x, w, bias, a, b, scale, row))
    for _ in range(3):                                # the same bits again, also where two tiles write a row
        assert torch.equal(y, o.linear_adapters(x, w, bias, bank, plan))
    xg = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(AdapterLinearFn.apply(xg, w, bias, a, b, scale, plan, 16), xg, dy)
    check(dx, *oracle2(dy, w.t(), None, b.transpose(1, 2), a.transpose(1, 2), scale, row))


@pytest.mark.parametrize("M", [2, 40, 300])
def test_what_is_left_of_products_that_cancel(M):
    """B = (1, -1) and two rows of A a hundredth apart: y is the small difference of two large ranks, all of it the adapter's."""
    o = ops()
    K, N = 256, 64
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(BF).to(DEV)
    a0 = torch.randn(1, 1, K, generator=g)
    a = torch.cat([a0, a0 + 0.01 * torch.randn(1, 1, K, generator=g)], 1).to(BF).to(DEV)
    b = torch.tensor([1.0, -1.0]).expand(1, N, 2).to(BF).to(DEV).contiguous()
    w = torch.zeros(N, K, device=DEV, dtype=BF)
    y = o.linear_adapters(x, w, None, o.AdapterBank(a, b, [1.0]), o.AdapterPlan([M], [0], DEV))
    want, tol = oracle2(x, w, None, a, b, [1.0], torch.zeros(M, device=DEV))
    check(y, want, tol)
    # (of the bound 264 2^-23 2 * 256 * 0.64 = 0.01 is the accumulation's; two ranks of size 16 rounded to bf16 would be off by up to 2^-8 16 = 0.06 each)


@pytest.mark.parametrize("r", [16, 32, 48, 72, 144, 256])
@pytest.mark.parametrize("K", [1984, 2048])
def test_a_row_that_two_tiles_write_gets_the_same_bits_from_both(r, K):
    """The last 256 x 256 tile is shifted inwards: rows 3844 .. 4095 are also the one's before.  Ranks in the K loop (all rows name one adapter) and behind it
    (the last rows name another) have to add up in the same order."""
    o = ops()
    M, N = 4100, 2056
    x, w, bias, a, b, scale, _ = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in problem([M], [0], K, N, r, BF, G=2))
    bank = o.AdapterBank(a, b, scale)
    o.launch_counts(reset=True)
    whole = o.linear_adapters(x, w, bias, bank, o.AdapterPlan([M], [0], DEV))
    assert o.launch_counts()["gemm_wide"] == 1
    mixed = o.AdapterPlan([M - 2, 2], [0, 1], DEV)
    for _ in range(4):
        assert torch.equal(o.linear_adapters(x, w, bias, bank, mixed)[:M - 2], whole[:M - 2])
