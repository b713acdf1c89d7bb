"""Infinities and NaN of an adapter's B and of u: every row gets what the formula gives it (0 inf = NaN, inf inf = inf, inf - inf = NaN), whatever
adapters its neighbours in a tile name.  Finite results: the tolerance of test_adapters_rounding_gpu.py."""
import pytest
import torch

from test_adapters_gpu import BF, DEV, F32, ops, problem
from test_adapters_rounding_gpu import oracle2

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dt,M,N,K", [(BF, 14, 64, 128), (BF, 150, 260, 128), (BF, 700, 1540, 200), (BF, 4100, 2052, 1984), (F32, 14, 64, 128),
                                      (F32, 150, 260, 128), (F32, 1100, 520, 132)])
@pytest.mark.parametrize("r", [5, 32, 72])
@pytest.mark.parametrize("alone", [False, True])
def test_rows_without_and_beyond_all_bounds_meet_an_adapter_that_is_not_finite(dt, M, N, K, r, alone):
    o = ops()
    lengths = [1, 2, 1, 1] + [M // 4, 1, M // 3]
    lengths.append(M - sum(lengths))
    ids = [0, 1, -1, 2, 1, 0, 2, -1]
    if alone:
        lengths, ids = [M], [1]
    x, w, bias, a, b, scale, row = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in problem(lengths, ids, K, N, r, dt, G=3))
    mine = (row == 1).nonzero().flatten()
    zero, huge = mine[0::5], mine[1::5]                    # u = 0: padding rows;  u[2] overflows
    x[:, 0], w[:, 0], a[:, :, 0] = 0, 0, 0
    x[zero] = 0
    want, tol = oracle2(x, w, bias, a, b, scale, row)
    u = scale[1] * (x[mine].double() @ a[1].double().t())
    b[1, 5, 2], b[1, 7, 0], b[1, 9, 4], b[1, 11, 1], b[1, 11, 3] = INF, NAN, -INF, INF, -INF
    x[huge, 0], a[1, 2, 0] = 1e38, 1e38                    # (x reaches rank 2 of adapter 1 through its channel 0 alone)
    u[1::5, 2] = INF
    assert (u[2::5] != 0).all() and (u[0::5] == 0).all()
    for c in (5, 7, 9, 11):
        want[mine, c] = (u * b[1, c].double()).sum(1)
    want[huge] = u[1::5] @ b[1].double().t()
    special = ~torch.isfinite(want)
    y = o.linear_adapters(x, w, bias, o.AdapterBank(a, b, scale), o.AdapterPlan(lengths, ids, DEV)).double()
    assert torch.isnan(want[zero][:, [5, 7, 9, 11]]).all() and (want[huge, 5] == INF).any() and special[huge].all()
    same = (torch.isnan(y) & torch.isnan(want)) | (y == want)
    assert same[special].all(), (special & ~same).nonzero()[:8].tolist()
    ok = ((y - want).abs() <= tol)[~special]
    assert ok.all(), int((~ok).sum())


def test_an_infinite_input_gives_infinite_gradients():
    """dA of an adapter whose kept input holds an infinity, dB where dy holds one: v inf is an infinity, not the NaN of two parts of different signs."""
    o = ops()
    lengths, ids = [100, 1, 60], [1, -1, 0]
    for dt in (BF, F32):
        x, w, _, a, b, scale, _ = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in problem(lengths, ids, 64, 72, 6, dt))
        plan = o.AdapterPlan(lengths, ids, DEV)
        bank = o.AdapterBank(a, b, scale, backward=True)
        dy = torch.randn(161, 72, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV)
        _, ut = o.linear_adapters(x, w, None, bank, plan, slots=True)
        x[3, 5], dy[130, 9], dy[40, 2] = INF, -INF, NAN
        _, da, db = o.linear_adapters_bwd(dy, w, bank, plan, x=x, ut=ut)
        u = scale[0] * (x[101:].double() @ a[0].double().t())
        # row 3's v is finite and not zero: +-inf in channel 5 of its adapter's dA; row 130's and row 40's v are not finite: all of their dA
        v = scale[1] * (dy[:100].double() @ b[1].double())
        assert torch.isnan(v[40]).all() and torch.isnan(da[1]).all() and not torch.isfinite(da[0]).any()
        assert torch.equal(db[0, 9], -torch.sign(u[29]).to(dt) * INF) and torch.isnan(db[1, 2]).all()
        ok = torch.ones(2, 72, dtype=torch.bool, device=DEV)
        ok[0, 9] = ok[1, 2] = False
        assert torch.isfinite(db[ok]).all()
        dy[40, 2] = 0.5
        _, da, _ = o.linear_adapters_bwd(dy, w, bank, plan, x=x, ut=ut)
        v3 = scale[1] * (dy[3].double() @ b[1].double())
        assert torch.equal(da[1, :, 5], torch.sign(v3).to(dt) * INF)
        da[1, :, 5] = 0
        assert torch.isfinite(da[1]).all()
