"""Low-rank adapters of many requests beside a shared projection (ops.linear_adapters, autograd.AdapterLinearFn) against float64.

Tolerances, per output element, h = eps / 2 of the type:
  y      h |y|  (its rounding)  +  h sum_r |u_r| |B_r|  (u is rounded to the type)  +  n 2^-23 S  (float32 accumulation of n terms of total size S)
  dx     likewise with v;   dA:  h |dA| + h^2 sum |v| |x| + n 2^-23 S (v in two parts: 16 bits in bf16);   dB:  with |dy| |u|.
The typical error is checked besides: the final rounding is at most h relative, uniform, so the error's rms is below h / sqrt(3) of the result's rms
for normal data: < 0.75 h."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def ops():
    from more4d_amd import ops as o
    return o


def problem(lengths, ids, K, N, r, dtype, G=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    G = G or max(max(ids) + 1, 1)
    M = sum(lengths)
    x = torch.randn(M, K, generator=g).to(dtype)
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype)
    bias = torch.randn(N, generator=g).to(dtype)
    a = (torch.randn(G, r, K, generator=g) * K ** -0.5).to(dtype)
    b = (0.3 * torch.randn(G, N, r, generator=g)).to(dtype)
    scale = [0.5 + 0.25 * i for i in range(G)]
    row = torch.tensor([i for n, i in zip(lengths, ids) for _ in range(n)], dtype=torch.long)
    return x, w, bias, a, b, scale, row


def oracle(x, w, bias, a, b, scale, row):
    """(y, bound) in float64"""
    h = torch.finfo(x.dtype).eps / 2
    K, R = x.shape[1], a.shape[1]
    xd, wd = x.double(), w.double()
    y = xd @ wd.t()
    S = xd.abs() @ wd.abs().t()
    U = torch.zeros_like(y)
    if bias is not None:
        y = y + bias.double()
        S = S + bias.double().abs()
    for i in range(a.shape[0]):
        m = row == i
        u = scale[i] * (xd[m] @ a[i].double().t())
        y[m] += u @ b[i].double().t()
        U[m] = u.abs() @ b[i].double().abs().t()
        S[m] += abs(scale[i]) * (xd[m].abs() @ a[i].double().abs().t()) @ b[i].double().abs().t()
    return y, h * (y.abs() + U) * 1.02 + (K + R + 4) * 2.0 ** -23 * S


FORWARD = [
    # lengths, ids, K, N, r, dtype
    ([1], [0], 64, 64, 4, BF),
    ([1], [0], 8, 4, 1, BF),
    ([1, 1], [1, 0], 1536, 516, 16, BF),
    ([1] * 8, [3, 0, -1, 4, 1, 0, 2, 5], 520, 772, 32, BF),
    ([3, 0, 61], [0, 1, 1], 128, 128, 8, BF),
    ([64, 1, 63, 2], [2, -1, 0, 2], 264, 260, 12, BF),
    ([129, 0, 77, 300], [0, 0, -1, 1], 200, 132, 20, BF),
    ([255, 1, 256], [1, 0, 1], 448, 512, 64, BF),               # 256 x 256 tiles, whole
    ([300, 1, 212, 190], [1, 0, -1, 2], 192, 776, 48, BF),      # ... ragged in both directions (the last tiles are shifted inwards)
    ([1] * 600, [i % 5 - 1 for i in range(600)], 128, 520, 16, BF),      # every row another request, adapters interleaved
    ([513], [0], 64, 512, 130, BF),
    ([520], [-1], 64, 512, 16, BF),                             # nobody names an adapter
    ([16], [0], 40, 20, 100, BF),
    ([7, 9], [1, 0], 4096, 96, 16, BF),                         # at most 16 rows, several steps per wave, a ragged last one
    ([17, 1], [0, 1], 1000, 200, 16, BF),                       # K in slices
    ([100], [0], 2056, 260, 16, BF),
    ([400, 100], [0, 1], 72, 1540, 16, BF),
    ([1], [0], 4, 4, 1, F32),
    ([9], [0], 516, 36, 5, F32),
    ([150], [0], 1028, 132, 16, F32),
    ([5, 0, 60, 70], [1, 0, 0, -1], 132, 68, 7, F32),
    ([300, 290], [0, 1], 100, 260, 40, F32),
]


@pytest.mark.parametrize("case", range(len(FORWARD)))
def test_forward(case):
    o = ops()
    lengths, ids, K, N, r, dt = FORWARD[case]
    x, w, bias, a, b, scale, row = problem(lengths, ids, K, N, r, dt)
    plan = o.AdapterPlan(lengths, ids, DEV)
    bank = o.AdapterBank(a.to(DEV), b.to(DEV), scale)
    for bs in (bias, None):
        poison = torch.full((sum(lengths) * bank.R,), float("nan"), device=DEV, dtype=dt)      # u of rows without an adapter is never read
        del poison
        y = o.linear_adapters(x.to(DEV), w.to(DEV), bs.to(DEV) if bs is not None else None, bank, plan)
        want, tol = oracle(x, w, bs, a, b, scale, row)
        assert y.dtype == dt and y.shape == want.shape
        err = (y.cpu().double() - want).abs()
        assert (err <= tol).all(), (float((err / tol).max()), FORWARD[case])
    assert torch.equal(y, o.linear_adapters(x.to(DEV), w.to(DEV), None, bank, plan))      # the same bits again


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("M", [70, 600])
def test_strided_operands(M, dt):
    """x a column range of a fused activation, w a row range and a column range, out a column range; what lies beside is left as it was."""
    o = ops()
    K, N, r = 128, 512, 8
    lengths, ids = [M - 33, 33], [1, 0]
    x, w, bias, a, b, scale, row = problem(lengths, ids, K, N, r, dt)
    xb, wb, ob = (torch.full(s, float("nan"), device=DEV, dtype=dt) for s in ((M, 3 * K), (N + 2, 2 * K), (M, N + 64)))
    xb[:, K:2 * K], wb[1:-1, K:] = x.to(DEV), w.to(DEV)
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a.to(DEV), b.to(DEV), torch.tensor(scale))
    out = ob[:, 32:32 + N]
    assert o.linear_adapters(xb[:, K:2 * K], wb[1:-1, K:], bias.to(DEV), bank, plan, out=out) is out
    want, tol = oracle(x, w, bias, a, b, scale, row)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert torch.isnan(ob[:, :32]).all() and torch.isnan(ob[:, 32 + N:]).all()
    x3 = o.linear_adapters(x.to(DEV).view(2, M // 2, K), w.to(DEV), bias.to(DEV), bank, plan)
    assert x3.shape == (2, M // 2, N) and ((x3.view(M, N).cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("M", [12, 150, 640])
def test_a_row_that_is_not_finite_stays_alone(M):
    o = ops()
    lengths, ids = [M // 2, 0, M - M // 2], [1, 2, 0]
    x, w, bias, a, b, scale, row = problem(lengths, ids, 128, 512, 16, BF)
    x[3, 5], x[M - 2, 7] = float("inf"), float("nan")
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a.to(DEV), b.to(DEV), scale)
    y = o.linear_adapters(x.to(DEV), w.to(DEV), bias.to(DEV), bank, plan).cpu()
    bad = torch.zeros(M, dtype=torch.bool)
    bad[3] = bad[M - 2] = True
    assert not torch.isfinite(y[bad]).any() and torch.isfinite(y[~bad]).all()
    x[bad] = 0
    want, tol = oracle(x, w, bias, a, b, scale, row)
    assert ((y.double() - want).abs() <= tol)[~bad].all()


def values8(o, x):
    return o.act_dequant8(o.act_quant8(x.to(DEV)), torch.float32).cpu().double()


BACKWARD = [
    ([1], [0], 64, 64, 4, BF),
    ([1, 1, 0], [1, 0, 2], 72, 36, 3, BF),
    ([65, 1, 130], [0, -1, 1], 136, 196, 16, BF),
    ([700, 1, 260], [1, 0, 1], 256, 512, 24, BF),
    ([200, 1100], [-1, 0], 712, 200, 200, BF),
    ([1] * 130, [i % 4 - 1 for i in range(130)], 96, 64, 8, BF),
    ([530], [0], 512, 576, 96, BF),
    ([2000], [0], 128, 64, 16, BF),
    ([33, 0, 70], [1, 0, 0], 68, 52, 5, F32),
    ([520, 80], [0, 2], 132, 516, 33, F32),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("case", range(len(BACKWARD)))
def test_backward(case, bits):
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids, K, N, r, dt = BACKWARD[case]
    G = max(ids) + 2                                  # one adapter that nobody names: zero gradients
    x, w, bias, a, b, scale, row = problem(lengths, ids, K, N, r, dt, G=G)
    M = x.shape[0]
    dy = torch.randn(M, N, generator=torch.Generator().manual_seed(9)).to(dt)
    plan = o.AdapterPlan(lengths, ids, DEV)
    xg, ag, bg = (t.to(DEV).requires_grad_(True) for t in (x, a, b))
    y = AdapterLinearFn.apply(xg, w.to(DEV), bias.to(DEV), ag, bg, scale, plan, bits)
    want, tol = oracle(x, w, bias, a, b, scale, row)
    assert ((y.detach().cpu().double() - want).abs() <= tol).all()
    dx, da, db = torch.autograd.grad(y, (xg, ag, bg), dy.to(DEV))
    assert dx.dtype == da.dtype == db.dtype == dt and da.shape == a.shape and db.shape == b.shape
    # dx is the same operator on dy with W^T, B^T and A^T
    wdx, tdx = oracle(dy, w.t(), None, b.transpose(1, 2), a.transpose(1, 2), scale, row)
    assert ((dx.cpu().double() - wdx).abs() <= tdx).all()
    h = torch.finfo(dt).eps / 2
    xd, dyd = (values8(o, x) if bits == 8 else x.double()), dy.double()
    num = {"a": 0.0, "b": 0.0}
    den = {"a": 0.0, "b": 0.0}
    for i in range(G):
        m = row == i
        v, u = scale[i] * (dyd[m] @ b[i].double()), scale[i] * (x.double()[m] @ a[i].double().t())
        va, ua = abs(scale[i]) * (dyd[m].abs() @ b[i].double().abs()), abs(scale[i]) * (x.double()[m].abs() @ a[i].double().abs().t())
        n = int(m.sum())
        wa, wb = v.t() @ xd[m], dyd[m].t() @ u
        ta = 1.02 * h * (wa.abs() + h * v.abs().t() @ xd[m].abs()) + (n + N) * 2.0 ** -23 * (va.t() @ xd[m].abs())
        tb = 1.02 * h * (wb.abs() + h * dyd[m].abs().t() @ u.abs()) + (n + K) * 2.0 ** -23 * (dyd[m].abs().t() @ ua)
        ea, eb = (da[i].cpu().double() - wa).abs(), (db[i].cpu().double() - wb).abs()
        assert (ea <= ta).all() and (eb <= tb).all(), (i, float((ea / ta).max()), float((eb / tb).max()))
        num["a"] += float(ea.pow(2).sum()); den["a"] += float(wa.pow(2).sum())
        num["b"] += float(eb.pow(2).sum()); den["b"] += float(wb.pow(2).sum())
        if n == 0:
            assert (da[i] == 0).all() and (db[i] == 0).all()
    if dt == BF and M > 100:
        for k in num:
            assert (num[k] / den[k]) ** 0.5 < 0.75 * h, k
    y2 = AdapterLinearFn.apply(xg, w.to(DEV), bias.to(DEV), ag, bg, scale, plan, bits)
    for p, q in zip(torch.autograd.grad(y2, (xg, ag, bg), dy.to(DEV)), (dx, da, db)):
        assert torch.equal(p, q)                      # the same bits again: no order-dependent sums


def test_gradients_against_differences():
    """L = sum(y * c) is linear in x, in A and in B taken one at a time, so the central difference along a direction is exact for any step: step 1.
    What remains is y's own error (the forward bound, through c) and the gradient's."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [40, 1, 90], [1, -1, 0]
    x, w, bias, a, b, scale, row = problem(lengths, ids, 64, 72, 6, F32)
    g = torch.Generator().manual_seed(3)
    c = torch.randn(131, 72, generator=g)
    plan = o.AdapterPlan(lengths, ids, DEV)
    t = [v.to(DEV).requires_grad_(True) for v in (x, a, b)]

    def run(xx, aa, bb):
        return AdapterLinearFn.apply(xx, w.to(DEV), bias.to(DEV), aa, bb, scale, plan, 16)

    grads = torch.autograd.grad(run(*t), t, c.to(DEV))
    for k in range(3):
        d = torch.randn(t[k].shape, generator=g)
        up, dn = list(map(lambda v: v.detach(), t)), list(map(lambda v: v.detach(), t))
        up[k], dn[k] = (up[k].cpu() + d).to(DEV), (dn[k].cpu() - d).to(DEV)
        diff = ((run(*up).cpu().double() - run(*dn).cpu().double()) * c.double()).sum() / 2
        want = (grads[k].cpu().double() * d.double()).sum()
        bound = 0.0
        for v in (up, dn):
            _, tol = oracle(v[0].cpu(), w, bias, v[1].cpu(), v[2].cpu(), scale, row)
            bound += float((tol * c.double().abs()).sum()) / 2
        # the perturbed inputs are rounded once (2^-24 of their size): part of the same bound's order; the gradient's error likewise
        assert abs(float(diff - want)) <= 3 * bound, (k, float(diff), float(want), bound)


def test_run_together_training_step_of_a_feed_forward():
    """adapter projection -> GELU kept in 8 bits -> adapter projection, forward and backward as a training step runs them, against float64 on the kept
    values: the 8-bit checkpoints enter the gradients of A (through the kept inputs) and the activation's derivative, nothing else."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [200, 0, 77, 1], [0, 1, 1, -1]
    M, C, F = 278, 128, 320
    plan = o.AdapterPlan(lengths, ids, DEV)
    x, w1, b1, a1, c1, s1, row = problem(lengths, ids, C, F, 8, F32, seed=1)
    _, w2, b2, a2, c2, s2, _ = problem(lengths, ids, F, C, 16, F32, seed=2)
    dout = torch.randn(M, C, generator=torch.Generator().manual_seed(5))
    p = [t.to(DEV).requires_grad_(True) for t in (x, a1, c1, a2, c2)]
    pre = AdapterLinearFn.apply(p[0], w1.to(DEV), b1.to(DEV), p[1], p[2], s1, plan, 8)
    kept = o.act_quant8(pre.detach())
    hid = o.unary(pre.detach(), F32, act=2).requires_grad_(True)
    out = AdapterLinearFn.apply(hid, w2.to(DEV), b2.to(DEV), p[3], p[4], s2, plan, 8)
    dh, da2, dc2 = torch.autograd.grad(out, (hid, p[3], p[4]), dout.to(DEV))
    dpre = o.act_bwd8(dh, kept, 2)
    dx, da1, dc1 = torch.autograd.grad(pre, (p[0], p[1], p[2]), dpre)

    def merged(w, a, c, s):
        return [w.double() + s[i] * c[i].double() @ a[i].double() for i in range(2)] + [w.double()]

    W1, W2 = merged(w1, a1, c1, s1), merged(w2, a2, c2, s2)
    P, H, O, DH, DX = (torch.zeros(M, n, dtype=torch.float64) for n in (F, F, C, F, C))
    for i, k in ((0, 0), (1, 1), (-1, 2)):
        m = row == i
        P[m] = x.double()[m] @ W1[k].t() + b1.double()
    H = torch.nn.functional.gelu(P, approximate="tanh")
    v = o.act_dequant8(kept).cpu().double().requires_grad_(True)
    (dact,) = torch.autograd.grad(torch.nn.functional.gelu(v, approximate="tanh").sum(), v)
    for i, k in ((0, 0), (1, 1), (-1, 2)):
        m = row == i
        O[m] = H[m] @ W2[k].t() + b2.double()
        DH[m] = dout.double()[m] @ W2[k]
    DP = DH * dact
    x8, h8 = values8(o, x), values8(o, hid.detach().cpu())
    for i, k in ((0, 0), (1, 1), (-1, 2)):
        m = row == i
        DX[m] = DP[m] @ W1[k]
        if i >= 0:
            for got, want in ((da1[i], s1[i] * (DP[m] @ c1[i].double()).t() @ x8[m]), (dc1[i], s1[i] * DP[m].t() @ (x.double()[m] @ a1[i].double().t())),
                              (da2[i], s2[i] * (dout.double()[m] @ c2[i].double()).t() @ h8[m]),
                              (dc2[i], s2[i] * dout.double()[m].t() @ (H[m] @ a2[i].double().t()))):
                # float32 throughout; 400 terms per sum, values of size 1: 400 * 2^-23 of the largest entry, twice for the chained products
                assert (got.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()
    for got, want in ((out.detach(), O), (dx, DX), (dpre, DP)):
        assert (got.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.parametrize("M", [5, 300, 700])
def test_streams_and_graph_replay(M):
    """On a side stream, and captured: two graphs of the same plan and bank, replayed in turn with eager calls between."""
    o = ops()
    lengths, ids = [M - 3, 2, 1], [0, -1, 1]
    x, w, bias, a, b, scale, row = problem(lengths, ids, 128, 512, 16, BF)
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a.to(DEV), b.to(DEV), scale)
    w, bias = w.to(DEV), bias.to(DEV)
    xs = [x.to(DEV), x.flip(0).contiguous().to(DEV)]
    want = [o.linear_adapters(v, w, bias, bank, plan) for v in xs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = o.linear_adapters(xs[0], w, bias, bank, plan)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want[0])
    graphs = []
    for v in xs:
        buf = torch.zeros_like(v)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, ut, b8 = o.linear_adapters(buf, w, bias, bank, plan, keep8=True)
            ga = o.adapter_grad(ut, b8, plan, bank)
        graphs.append((g, buf, y, ga))
    for i in range(4):
        for k, (g, buf, y, ga) in enumerate(graphs):
            v = xs[(i + k) % 2]
            buf.copy_(v)
            g.replay()
            eager = o.adapter_grad(o.adapter_down(v, bank, plan, slots=True)[1], o.act_quant8(v), plan, bank)
            torch.cuda.synchronize()
            assert torch.equal(y, want[(i + k) % 2]) and torch.equal(ga, eager)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("K", [8, 40, 64, 200, 712])
def test_the_pass_that_reads_x_writes_the_same_codes(K, dt):
    """linear_adapters(keep8=True) against act_quant8 on the rows that name an adapter, infinities and NaN among them."""
    o = ops()
    lengths, ids = [70, 3, 150, 33], [1, -1, 0, 1]
    x, w, bias, a, b, scale, row = problem(lengths, ids, K, 64, 8, dt)
    x = x * torch.exp(3 * torch.randn(1, K, generator=torch.Generator().manual_seed(4))).to(dt)
    x[5, 3], x[100, 7], x[101, 0] = float("inf"), float("nan"), 3e38
    xd = x.to(DEV)
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a.to(DEV), b.to(DEV), scale)
    y, ut, x8 = o.linear_adapters(xd, w.to(DEV), bias.to(DEV), bank, plan, keep8=True)
    ref = o.act_quant8(xd)
    on = (row >= 0).to(DEV)
    assert torch.equal(x8.codes[on], ref.codes[on]) and torch.equal(x8.exps[on], ref.exps[on])
    y2, ut2 = o.linear_adapters(xd, w.to(DEV), bias.to(DEV), bank, plan, slots=True)
    assert torch.equal(y.nan_to_num(0), y2.nan_to_num(0)) and torch.equal(ut.nan_to_num(0), ut2.nan_to_num(0))
    u, ut3 = o.adapter_down(xd, bank, plan, slots=True)
    assert torch.equal(ut3.nan_to_num(0), ut.nan_to_num(0))
    slot = torch.tensor(tables_slot_row(plan))
    # [slot / 16][rank / 32][part][rank % 32 + 32 * (slot % 16 / 8)][slot % 8] -> [part][slot][rank]
    v = ut.cpu().view(len(slot) // 16, ut.shape[1], -1, 2, 32, 8).permute(2, 0, 3, 5, 1, 4).reshape(ut.shape[2], len(slot), -1)
    assert (v[:, slot < 0] == 0).all() and (v[:, slot >= 0][..., 8:].nan_to_num(0) == 0).all()
    on_slot = v[:, slot >= 0][..., :u.shape[1]].nan_to_num(0).double()
    uu = u.cpu()[slot[slot >= 0].long()].nan_to_num(0).double()
    assert torch.equal(on_slot[0], uu)
    if dt == BF:                                       # the second part: what the first one's rounding left, at most half of its last bit
        fin = uu.abs() < 1e38
        assert (on_slot[1].abs()[fin] <= uu.abs()[fin] * torch.finfo(BF).eps / 2 + 1e-38).all() and on_slot[1].abs().max() > 0


def tables_slot_row(plan):
    o = (plan.args.slot_row - plan.table.data_ptr()) // 4
    return plan.table.cpu().tolist()[o:o + 64 * plan.n_pieces]


def test_no_rows_and_refusals():
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    x, w, bias, a, b, scale, _ = problem([8], [0], 64, 32, 4, BF)
    x, w, bias, a, b = (t.to(DEV) for t in (x, w, bias, a, b))
    bank = o.AdapterBank(a, b, scale)
    plan = o.AdapterPlan([8], [0], DEV)
    empty = o.AdapterPlan([0, 0], [0, 1], DEV)
    assert o.linear_adapters(x[:0], w, bias, bank, empty).shape == (0, 32)
    y = AdapterLinearFn.apply(x[:0].requires_grad_(True), w, bias, a.clone().requires_grad_(True), b, scale, empty, 8)
    y.sum().backward()
    for bad in (lambda: o.linear_adapters(x[:7], w, bias, bank, plan), lambda: o.linear_adapters(x[:0], w, bias, bank, plan),
                lambda: o.linear_adapters(x, w[:, :32], bias, bank, plan), lambda: o.linear_adapters(x, w[:16], bias[:16], bank, plan),
                lambda: o.linear_adapters(x, w, bias[:8], bank, plan), lambda: o.linear_adapters(x, w, bias, bank, o.AdapterPlan([8], [1], DEV)),
                lambda: o.linear_adapters(x, w, bias, bank, plan, out=torch.empty(8, 16, device=DEV, dtype=BF)),
                lambda: bank.transposed(),
                lambda: o.AdapterBank(a, b[:, :, :2], scale), lambda: o.AdapterBank(a, b, [1.0, 2.0]),
                lambda: AdapterLinearFn.apply(x, w, bias, a, b, scale, plan, 4),
                lambda: AdapterLinearFn.apply(x, w.clone().requires_grad_(True), bias, a, b, scale, plan, 8)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: o.linear_adapters(x.float(), w, bias, bank, plan), lambda: o.AdapterBank(a, b.float(), scale),
                lambda: o.linear_adapters(x.float(), w.float(), None, bank, plan)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(o._lib.More4DHipError):             # rows that are not 16-byte aligned
        o.linear_adapters(torch.zeros(8, 65, device=DEV, dtype=BF)[:, 1:], w, bias, bank, plan)
