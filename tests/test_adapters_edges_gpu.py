"""Low-rank adapters beside a shared projection: adapters that are not finite, the largest tiles, long offsets, partial gradients, captured steps.
Tolerances as in test_adapters_gpu.py (its oracle, evaluated in float64 on the GPU for the larger sizes)."""
import pytest
import torch

from test_adapters_gpu import BF, DEV, F32, oracle, ops, problem

pytestmark = pytest.mark.gpu


def on_gpu(*ts):
    return [t.to(DEV) if isinstance(t, torch.Tensor) else t for t in ts]


WIDE = (4100, 2052, 1984)      # M, N, K: the size rule sends it to the 256 x 256 tiles, the last ones shifted inwards, an odd number of K tiles


@pytest.mark.parametrize("dt,M,N,K", [(BF, 14, 64, 128), (BF, 150, 260, 128), (BF, 700, 1540, 200), (BF, *WIDE), (F32, 14, 64, 128), (F32, 150, 260, 128),
                                      (F32, 1100, 520, 132)])
@pytest.mark.parametrize("r", [5, 72])
def test_an_adapter_that_is_not_finite_stays_with_its_rows(dt, M, N, K, r):
    """B of one adapter holds infinities and a NaN: its rows get what the formula says, every other row what it gets without."""
    o = ops()
    lengths = [1, 2, 1, 1] + [M // 4, 1, M // 3]
    lengths.append(M - sum(lengths))
    ids = [0, 1, -1, 2, 1, 0, 2, -1]
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, K, N, r, dt))
    b[1, 5, 2], b[1, 7, 0], b[1, 9, 4] = float("inf"), float("nan"), -float("inf")
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale)
    y = o.linear_adapters(x, w, bias, bank, plan).double()
    u, _ = o.adapter_down(x, bank, plan)
    clean = b.clone()
    clean[1, 5, 2] = clean[1, 7, 0] = clean[1, 9, 4] = 0
    want, tol = oracle(x, w, bias, a, clean, scale, row)
    mine = row == 1
    ok = ((y - want).abs() <= tol)
    ok[mine, 5] = y[mine, 5] == float("inf") * u[mine, 2].double()
    ok[mine, 7] = torch.isnan(y[mine, 7])
    ok[mine, 9] = y[mine, 9] == -float("inf") * u[mine, 4].double()
    assert (u[mine][:, [2, 4]] != 0).all()
    assert ok.all(), (~ok).nonzero()[:8].tolist()


def test_changes_between_forward_and_backward():
    """A scale tensor that wants a gradient is refused; x, W or scale changed in place between the passes raises; a and b may change (laid out)."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [30, 3, 40], [1, -1, 0]
    x, w, bias, a, b, scale, _ = on_gpu(*problem(lengths, ids, 64, 72, 4, BF))
    plan, s = o.AdapterPlan(lengths, ids, DEV), torch.tensor(scale, device=DEV)
    dy = torch.randn(73, 72, device=DEV).to(BF)
    with pytest.raises(ValueError):
        AdapterLinearFn.apply(x, w, bias, a, b, s.clone().requires_grad_(True), plan, 8)
    with pytest.raises(ValueError):                       # rows padded beyond the adapters' K: serving only
        AdapterLinearFn.apply(x, w, bias, a[:, :, :60], b, s, plan, 8)

    def run(change):
        xx, ww, ss, aa, bb = x.clone(), w.clone(), s.clone(), a.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = AdapterLinearFn.apply(xx, ww, bias, aa, bb, ss, plan, 16)
        with torch.no_grad():
            change(xx, ww, ss, aa, bb)
        return torch.autograd.grad(y, (aa, bb), dy)

    want = run(lambda *t: None)
    for i in range(3):
        with pytest.raises(RuntimeError):
            run(lambda *t: t[i].mul_(2))
    for i in (3, 4):
        for p, q in zip(run(lambda *t: t[i].mul_(2)), want):
            assert torch.equal(p, q)
