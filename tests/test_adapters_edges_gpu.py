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


def check(y, want, tol):
    err = (y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("lengths,ids,r", [
    ([4100], [0], 16),                                      # one adapter, ranks behind the K loop
    ([4100], [0], 64),                                      # ... as one more K tile
    ([4100], [0], 144),                                     # ... as two and a remainder
    ([256, 2048, 1796], [2, 0, 1], 72),                     # whole tiles of each, the shifted last one of one adapter
    ([1000, 1, 2000, 0, 1099], [1, 0, -1, 2, 1], 64),       # tiles of several, tiles of none
    ([1] * 300 + [3800], [i % 7 - 1 for i in range(300)] + [0], 8),
])
@pytest.mark.parametrize("K", [1984, 2048])
def test_the_largest_tiles(lengths, ids, r, K):
    o = ops()
    M, N, _ = WIDE
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, K, N, r, BF))
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale)
    out = torch.full((M + 1, N + 4), float("nan"), device=DEV, dtype=BF)
    o.launch_counts(reset=True)
    y = o.linear_adapters(x, w, bias, bank, plan, out=out[:M, :N])
    assert o.launch_counts()["gemm_wide"] == 1
    check(y, *oracle(x, w, bias, a, b, scale, row))
    assert torch.isnan(out[M]).all() and torch.isnan(out[:, N:]).all()
    assert torch.equal(y, o.linear_adapters(x, w, bias, bank, plan))


def test_offsets_beyond_32_bits():
    """x of 2^31 + elements: its last rows, which alone name adapters with those at the front, in every pass that addresses rows."""
    o = ops()
    K, N, r, M = 4096, 64, 16, (1 << 19) + 700
    lengths, ids = [200, M - 500, 300], [0, -1, 1]
    _, w, bias, a, b, scale, _ = on_gpu(*problem([1, 1], [0, 1], K, N, r, BF))
    x = torch.zeros(M, K, device=DEV, dtype=BF)
    x[:200].normal_()
    x[-300:].normal_()
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale)
    y, ut, x8 = o.linear_adapters(x, w, bias, bank, plan, keep8=True)
    ends = torch.cat([torch.arange(200), torch.arange(M - 300, M)]).to(DEV)
    rows, xe = torch.cat([torch.zeros(200), torch.ones(300)]).long().to(DEV), x[ends]
    check(y[ends], *oracle(xe, w, bias, a, b, scale, rows))
    assert torch.equal(y[200:-300], bias.expand(M - 500, N))
    small = o.AdapterPlan([200, 300], [0, 1], DEV)
    ref8 = o.act_quant8(xe)
    assert torch.equal(x8.codes[ends], ref8.codes) and torch.equal(x8.exps[ends], ref8.exps)
    big, few = o.adapter_grad(ut, x8, plan, bank), o.adapter_grad(o.adapter_down(xe, bank, small, slots=True)[1], xe, small, bank)
    assert torch.equal(o.adapter_grad(ut, x, plan, bank), few)
    h = torch.finfo(BF).eps / 2
    v8 = o.act_dequant8(ref8).double()
    u = o.adapter_down(xe, bank, small)[0].double()[:, :r]
    for g in range(2):                                     # (u rounded to bf16 once instead of kept to 16 bits: h of every term more)
        want = u[rows == g].t() @ v8[rows == g]
        tol = h * want.abs() + (2 * h + 500 * 2.0 ** -23) * (u[rows == g].abs().t() @ v8[rows == g].abs())
        check(big[g], want, tol)
    q = o.act_quant8(x)
    assert torch.equal(q.codes[ends], ref8.codes) and not q.codes[200:-300].any()
    assert torch.equal(o.act_dequant8(q)[ends], o.act_dequant8(ref8))
    t = o.act_dequant8_t(q, act=1)
    assert t.shape[1] >= M and torch.equal(t[:, ends], o.act_dequant8(ref8, act=1).t().contiguous()) and not t[:, M:].any()
    del t, q
    x.fill_(1.0)
    assert torch.equal(o.act_bwd8(x, x8, 2, out=x)[ends], o.act_bwd8(torch.ones_like(xe), ref8, 2))


def test_a_long_output():
    """out of 2^31 + elements: the tiles' stores at its end."""
    o = ops()
    K, r, N, M = 64, 16, 32768, 65536 + 300
    lengths, ids = [M - 300, 300], [0, 1]
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, K, N, r, BF))
    y = o.linear_adapters(x, w, bias, o.AdapterBank(a, b, scale), o.AdapterPlan(lengths, ids, DEV))
    for sl in (slice(0, 300), slice(M // 2, M // 2 + 300), slice(M - 600, M)):
        check(y[sl], *oracle(x[sl], w, bias, a, b, scale, row[sl]))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("wants", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("N", [64, 68])
def test_some_of_the_gradients(wants, dt, N):
    """Any of x, A, B may not be trained, bias may be missing, dy may be an expanded scalar or a column range."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [70, 2, 40], [1, -1, 0]
    x, w, _, a, b, scale, _ = on_gpu(*problem(lengths, ids, 72, N, 6, dt))
    plan = o.AdapterPlan(lengths, ids, DEV)
    wide = torch.randn(112, 3 * N, device=DEV).to(dt)
    for bits in (8, 16):
        for dy in (wide[:, N:2 * N], torch.ones(1, device=DEV, dtype=dt).expand(112, N)):
            t = [v.clone().requires_grad_(True) for v in (x, a, b)]
            full = torch.autograd.grad(AdapterLinearFn.apply(t[0], w, None, t[1], t[2], scale, plan, bits), t, dy.contiguous())
            t = [v.clone().requires_grad_(bool(k)) for v, k in zip((x, a, b), wants)]
            some = torch.autograd.grad(AdapterLinearFn.apply(t[0], w, None, t[1], t[2], scale, plan, bits), [v for v in t if v.requires_grad], dy)
            for p, q in zip(some, [f for f, k in zip(full, wants) if k]):
                assert torch.equal(p, q)


@pytest.mark.parametrize("dt", [BF, F32])
def test_nobody_names_an_adapter(dt):
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    x, w, bias, a, b, scale, row = on_gpu(*problem([90], [-1], 64, 68, 6, dt))
    plan = o.AdapterPlan([90], [-1], DEV)
    t = [v.requires_grad_(True) for v in (x, a, b)]
    y = AdapterLinearFn.apply(*t[:1], w, bias, *t[1:], scale, plan, 8)
    dy = torch.randn(90, 68, device=DEV).to(dt)
    dx, da, db = torch.autograd.grad(y, t, dy)
    check(y.detach(), *oracle(x.detach(), w, bias, a.detach(), b.detach(), scale, row))
    check(dx, *oracle(dy, w.t(), None, b.detach().transpose(1, 2), a.detach().transpose(1, 2), scale, row))
    assert not da.any() and not db.any()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("M", [9, 333])
def test_the_largest_rank(dt, M):
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [M - 3, 3], [1, 0]
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, 520, 264, 512, dt))
    plan = o.AdapterPlan(lengths, ids, DEV)
    t = [v.requires_grad_(True) for v in (x, a, b)]
    y = AdapterLinearFn.apply(*t[:1], w, bias, *t[1:], scale, plan, 16)
    dy = torch.randn(M, 264, device=DEV).to(dt)
    dx, da, db = (g.double() for g in torch.autograd.grad(y, t, dy))
    x, a, b = (v.detach() for v in t)
    check(y.detach(), *oracle(x, w, bias, a, b, scale, row))
    check(dx, *oracle(dy, w.t(), None, b.transpose(1, 2), a.transpose(1, 2), scale, row))
    h = torch.finfo(dt).eps / 2
    for g in range(2):
        m = row == g
        v, u = scale[g] * dy[m].double() @ b[g].double(), scale[g] * x[m].double() @ a[g].double().t()
        va, ua = scale[g] * dy[m].double().abs() @ b[g].double().abs(), scale[g] * x[m].double().abs() @ a[g].double().abs().t()
        for got, p, q, s, n in ((da[g], v, x[m].double(), va, 264), (db[g].t(), u, dy[m].double(), ua, 520)):
            want = p.t() @ q
            check(got, want, 1.02 * h * (want.abs() + h * p.abs().t() @ q.abs()) + (M + n) * 2.0 ** -23 * (s.t() @ q.abs()))


def test_a_captured_training_step():
    """Forward and backward of two layers in one graph, replayed with other inputs and eager steps of the same leaves between."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [200, 1, 99], [1, -1, 0]
    x, w1, _, a1, b1, scale, _ = on_gpu(*problem(lengths, ids, 128, 256, 8, BF))
    _, w2, _, a2, b2, _, _ = on_gpu(*problem(lengths, ids, 256, 128, 8, BF, seed=1))
    plan, s = o.AdapterPlan(lengths, ids, DEV), torch.tensor(scale, device=DEV)
    leaves = [v.requires_grad_(True) for v in (a1, b1, a2, b2)]

    def step(xx, dy):
        xx = xx.detach().requires_grad_(True)
        y = AdapterLinearFn.apply(AdapterLinearFn.apply(xx, w1, None, a1, b1, s, plan, 8), w2, None, a2, b2, s, plan, 16)
        return torch.autograd.grad(y, [xx] + leaves, dy)

    gen = torch.Generator().manual_seed(1)
    data = [(torch.randn(300, 128, generator=gen).to(BF).to(DEV), torch.randn(300, 128, generator=gen).to(BF).to(DEV)) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*data[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    xs, ds = (torch.zeros_like(v) for v in data[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(xs, ds)
    for i in range(5):
        xs.copy_(data[i % 3][0])
        ds.copy_(data[i % 3][1])
        g.replay()
        eager = step(*data[i % 3])
        torch.cuda.synchronize()
        for p, q in zip(out, eager):
            assert torch.equal(p, q)


def test_two_streams_at_once():
    """Calls that share plan and bank, on two streams without waiting for each other."""
    o = ops()
    lengths, ids = [700, 1, 300], [1, -1, 0]
    x, w, bias, a, b, scale, _ = on_gpu(*problem(lengths, ids, 512, 512, 16, BF))
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale, backward=True)
    xs = [x, x.flip(0).contiguous()]

    def run(v):
        y, ut, x8 = o.linear_adapters(v, w, bias, bank, plan, keep8=True)
        return (y,) + o.linear_adapters_bwd(y, w, bank, plan, x=x8, ut=ut)

    want = [run(v) for v in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(xs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            for p, q in zip(r, want[k]):
                assert torch.equal(p, q)


@pytest.mark.parametrize("dt,M,N,K,r", [(BF, 200, 260, 1000, 16), (BF, 700, 1540, 200, 40), (BF, 1500, 2052, 256, 64), (F32, 300, 516, 260, 20), (F32, 1200, 1028, 64, 8)])
def test_interleaved_requests(dt, M, N, K, r):
    """One-row requests of 24 adapters, some of none: tiles of rows in order of their adapters, K slices among them; rows of a wider tensor."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    ids = [(i * 7) % 25 - 1 for i in range(M)]
    x, w, bias, a, b, scale, row = on_gpu(*problem([1] * M, ids, K, N, r, dt))
    plan, bank = o.AdapterPlan([1] * M, ids, DEV), o.AdapterBank(a, b, scale)
    assert plan.args.row_order
    out = torch.full((M, N + 8), float("nan"), device=DEV, dtype=dt)
    y = o.linear_adapters(x, w, bias, bank, plan, out=out[:, :N])
    check(y, *oracle(x, w, bias, a, b, scale, row))
    assert torch.isnan(out[:, N:]).all()
    t = [v.requires_grad_(True) for v in (x, a, b)]
    y = AdapterLinearFn.apply(t[0], w, None, t[1], t[2], scale, plan, 16)
    dy = torch.randn(M, N, device=DEV).to(dt)
    dx, da, db = torch.autograd.grad(y, t, dy)
    x, a, b = (v.detach() for v in t)
    check(dx, *oracle(dy, w.t(), None, b.transpose(1, 2), a.transpose(1, 2), scale, row))
    by = sorted(range(M), key=lambda i: (ids[i], i))
    srt = o.AdapterPlan([1] * M, [ids[i] for i in by], DEV)
    t = [v.clone().requires_grad_(True) for v in (x[by], a, b)]
    ys = AdapterLinearFn.apply(t[0], w, None, t[1], t[2], scale, srt, 16)
    _, da2, db2 = torch.autograd.grad(ys, t, dy[by])
    assert torch.equal(da, da2) and torch.equal(db, db2)              # the same slots, so the same sums


@pytest.mark.parametrize("M,lengths,ids", [(4400, [4400], [0]), (4400, [3000, 1, 900, 0, 400, 99], [1, 0, -1, 0, 2, 1]), (3850, [3838, 1, 6, 5], [0, 1, -1, 2]),
                                           (3841, [3841], [-1]), (4000, [3840, 160], [-1, 0])])
@pytest.mark.parametrize("r", [16, 64])
def test_whole_rounds_of_the_largest_tiles_and_the_rows_behind(M, lengths, ids, r):
    o = ops()
    N, K = 4100, 1024
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, K, N, r, BF))
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale) if max(ids) >= 0 else o.AdapterBank(a[:1], b[:1], scale[:1])
    out = torch.full((M + 1, N + 4), float("nan"), device=DEV, dtype=BF)
    o.launch_counts(reset=True)
    y = o.linear_adapters(x, w, bias, bank, plan, out=out[:M, :N])
    n = o.launch_counts()
    if max(ids) >= 0:
        assert n["gemm_wide"] == 1 and n["gemm_generic"] == 1
    check(y, *oracle(x, w, bias, a, b, scale, row))
    assert torch.isnan(out[M]).all() and torch.isnan(out[:, N:]).all()


@pytest.mark.parametrize("lengths,ids,K,N", [([512, 77, 1, 0, 226, 131, 39], [0, 2, 1, 1, -1, 2, 3], 4096, 5124), ([300], [0], 4096, 5120),
                                             ([1] * 986, [i % 9 - 1 for i in range(986)], 1024, 5120), ([2900, 100], [1, 0], 8960, 1540)])
def test_tiles_of_192_columns(lengths, ids, K, N):
    """Shapes that the size rule sends to the 128 x 192 tiles: whole K, slices of K, rows in order of their adapters, a ragged last column tile."""
    o = ops()
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, K, N, 12, BF))
    M = x.shape[0]
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale)
    out = torch.full((M + 1, N + 8), float("nan"), device=DEV, dtype=BF)
    y = o.linear_adapters(x, w, bias, bank, plan, out=out[:M, :N])
    check(y, *oracle(x, w, bias, a, b, scale, row))
    assert torch.isnan(out[M]).all() and torch.isnan(out[:, N:]).all()
    assert torch.equal(y, o.linear_adapters(x, w, bias, bank, plan))


def test_rows_far_apart():
    """Row strides whose 31-fold passes 32 bits in bytes: not for the 256 x 256 tiles, which the shape would go to otherwise."""
    o = ops()
    M, N, K, ld = 512, 30720, 1024, 70_000_000
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 72 GB")
    lengths, ids = [300, 212], [1, 0]
    x, w, bias, a, b, scale, row = on_gpu(*problem(lengths, ids, K, N, 16, BF))
    far = torch.empty((M - 1) * ld + K, device=DEV, dtype=BF).as_strided((M, K), (ld, 1))
    far.copy_(x)
    plan, bank = o.AdapterPlan(lengths, ids, DEV), o.AdapterBank(a, b, scale)
    o.launch_counts(reset=True)
    y = o.linear_adapters(far, w, bias, bank, plan)
    assert o.launch_counts()["gemm_wide"] == 0
    check(y, *oracle(x, w, bias, a, b, scale, row))
    o.launch_counts(reset=True)
    check(o.linear_adapters(x, w, bias, bank, plan), *oracle(x, w, bias, a, b, scale, row))
    assert o.launch_counts()["gemm_wide"] == 1
    del far
    torch.cuda.empty_cache()


def test_a_second_derivative_is_refused():
    """The backward's kernels leave no graph: a gradient of a gradient raises, it does not come out without their part."""
    from more4d_amd.autograd import AdapterLinearFn
    o = ops()
    lengths, ids = [30, 3, 40], [1, -1, 0]
    x, w, bias, a, b, scale, _ = on_gpu(*problem(lengths, ids, 64, 72, 4, BF))
    x = x.requires_grad_(True)
    y = AdapterLinearFn.apply(x, w, bias, a.requires_grad_(True), b, scale, o.AdapterPlan(lengths, ids, DEV), 16)
    (dx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        (dx.float().square().sum() + x.float().square().sum()).backward()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows,K,per", [(300, 8960, 9), (1600, 8192, 13), (21800, 5120, 27)])
def test_codes_of_slices_that_begin_on_odd_chunks(rows, K, per, dt):
    """Slices of K of an odd number of 64-channel chunks: the exponents of a row, two bytes a chunk, meet in one dword from two workgroups."""
    from more4d_amd import _lib
    o = ops()
    x, w, bias, a, b, scale, _ = on_gpu(*problem([rows], [0], K, 64, 16, dt))
    x *= torch.exp(3 * torch.randn(1, K, generator=torch.Generator().manual_seed(4))).to(dt).to(DEV)
    x[5, 3], x[rows - 1, K - 1] = float("inf"), float("nan")
    plan, bank = o.AdapterPlan([rows], [0], DEV), o.AdapterBank(a, b, scale)
    slices = _lib.load().m4d_adapter_down_workspace(plan.args, K, bank.R, 1) // (plan.n_pieces * 32 * 64)
    assert -(-(K // 64) // slices) == per and per % 2 == 1
    _, ut, x8 = o.linear_adapters(x, w, bias, bank, plan, keep8=True)
    ref = o.act_quant8(x)
    assert torch.equal(x8.codes, ref.codes) and torch.equal(x8.exps, ref.exps)
    assert torch.equal(ut.nan_to_num(0), o.adapter_down(x, bank, plan, slots=True)[1].nan_to_num(0))
