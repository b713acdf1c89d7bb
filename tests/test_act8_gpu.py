"""Activations kept in 8 bits (m4d_act_quant8 and its readers) against their definition in 64 bits.

Codes and steps are exact (the step is a power of two), so they are compared for equality.  Tolerances of the activation readers: one rounding to the
output type, |want| * eps / 2, plus the float32 evaluation of the function: its argument's rounding (a few 2^-24 times the argument, at most 32,
times the function's slope, at most 1.13) and two hardware operations of 2^-23: 32 * 4 * 2^-24 + 2^-22 < 1e-5, on values of magnitude 1."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float32]


def ops():
    from more4d_amd import ops as o
    return o


def oracle_codes(x):
    """float64 [rows, C] -> (codes int, exps int, values float64): one block at a time, the exponent by search."""
    rows, C = x.shape
    nb = -(-C // 32)
    codes = torch.zeros(rows, nb * 32, dtype=torch.int64)
    exps = torch.zeros(rows, nb, dtype=torch.int64)
    vals = torch.empty(rows, C, dtype=torch.float64)
    for j in range(nb):
        b = x[:, 32 * j:32 * j + 32]
        bad = ~torch.isfinite(b).all(dim=1)
        top = torch.where(bad[:, None], torch.zeros_like(b), b).abs().amax(dim=1)
        e = torch.full((rows,), -126, dtype=torch.float64)
        while True:
            low = (127.0 * torch.exp2(e) < top) & (e < 121)
            if not low.any():
                break
            e = torch.where(low, e + 1, e)
        q = (torch.where(bad[:, None], torch.zeros_like(b), b) / torch.exp2(e)[:, None]).round().clamp(-127, 127)
        codes[:, 32 * j:32 * j + b.shape[1]] = q.long()
        exps[:, j] = torch.where(bad, torch.full_like(e, 255), e + 127).long()
        v = q * torch.exp2(e)[:, None]
        vals[:, 32 * j:32 * j + b.shape[1]] = torch.where(bad[:, None], torch.full_like(v, float("nan")), v)
    return codes, exps, vals


def activations(rows, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g) * torch.exp(2 * torch.randn(1, C, generator=g)) * torch.exp(torch.randn(rows, 1, generator=g))
    return x.to(dtype)


SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 40), (7, 1536), (129, 200), (64, 1000), (513, 260), (1, 13824)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", SHAPES)
def test_codes_equal_their_definition(rows, C, dtype):
    o = ops()
    x = activations(rows, C, dtype)
    a8 = o.act_quant8(x.to(DEV))
    codes, exps, vals = oracle_codes(x.double())
    assert torch.equal(a8.exps.cpu().long(), exps)
    assert torch.equal(a8.codes.cpu().long(), codes)
    for dt in DTYPES:
        assert torch.equal(o.act_dequant8(a8, dt).cpu().double(), vals)      # 7-bit codes times a power of two: exact in both types
    assert o.act_dequant8(a8).dtype == dtype
    assert a8.nbytes() == rows * -(-C // 32) * 33


def test_codes_at_the_borders_of_the_format():
    """Zero blocks, ties, max = 127 * 2^e exactly and one step above, subnormal and huge values, infinities and NaN in one block only."""
    o = ops()
    blocks = []
    base = torch.linspace(-1, 1, 32, dtype=torch.float64)
    blocks.append(torch.zeros(32, dtype=torch.float64))
    blocks.append(-torch.zeros(32, dtype=torch.float64))
    for top in (127.0, 127.0 * 2.0 ** -20, 127.5, 128.0, 64.0, 63.5):
        b = base * top
        b[0] = top
        blocks.append(b)
    blocks.append((torch.arange(32, dtype=torch.float64) - 16) + 0.5)          # with max 127: exact ties
    blocks[-1][0] = 127.0
    blocks.append(base * 2.0 ** -130)                                          # float32 subnormals
    blocks.append(base * 2.0 ** -149 * 3)
    blocks.append(base * 3.38e38)                                              # e is capped, codes saturate
    for v in (float("inf"), float("-inf"), float("nan")):
        b = base.clone()
        b[5] = v
        blocks.append(b)
    blocks.append(base)
    x = torch.cat(blocks).view(1, -1).float()
    for xx in (x, x.bfloat16(), torch.cat([x, x.flip(1)]).contiguous()):
        a8 = o.act_quant8(xx.to(DEV))
        codes, exps, vals = oracle_codes(xx.double())
        assert torch.equal(a8.exps.cpu().long(), exps) and torch.equal(a8.codes.cpu().long(), codes)
        got = o.act_dequant8(a8, torch.float32).cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(vals)) and torch.equal(got.nan_to_num(0.0), vals.nan_to_num(0.0))
        assert torch.isfinite(got[~torch.isnan(vals)]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_a_wider_tensor(dtype):
    """A column range of a wider matrix (fused projections), 3-D inputs, and a start that is not 16-byte aligned; what lies beside is untouched."""
    o = ops()
    wide = activations(37, 480, dtype).to(DEV)
    for lo, hi in ((0, 160), (160, 320), (3, 100), (479, 480)):
        x = wide[:, lo:hi]
        a8 = o.act_quant8(x)
        codes, exps, vals = oracle_codes(x.cpu().double())
        assert torch.equal(a8.codes.cpu().long(), codes) and torch.equal(a8.exps.cpu().long(), exps)
        out = torch.full_like(wide, 7.0)
        o.act_dequant8(a8, out=out[:, lo:hi])
        assert torch.equal(out[:, lo:hi].cpu().double(), vals)
        out[:, lo:hi] = 7.0
        assert (out == 7.0).all()
        d = torch.full_like(wide, 7.0)
        o.act_bwd8(x, a8, 2, out=d[:, lo:hi])
        assert torch.equal(d[:, lo:hi], o.act_bwd8(x.contiguous(), a8, 2))
        d[:, lo:hi] = 7.0
        assert (d == 7.0).all()
    x3 = wide.view(37, 4, 120)
    assert torch.equal(o.act_dequant8(o.act_quant8(x3)), o.act_dequant8(o.act_quant8(x3.reshape(148, 120))).view(37, 4, 120))
    again = o.act_quant8(wide)
    other = o.act_quant8(wide.flip(0).contiguous(), out=again)
    assert other is again and torch.equal(o.act_dequant8(again).cpu().double(), oracle_codes(wide.flip(0).cpu().double())[2])


def act64(v, act):
    v = v.clone().requires_grad_(True)
    h = v * torch.sigmoid(v) if act == 1 else 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))) if act == 2 else \
        0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    (d,) = torch.autograd.grad(h.sum(), v)
    return h.detach(), d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("rows,C", [(1, 8), (3, 33), (66, 130), (129, 256), (700, 264)])
def test_use_in_the_backward(rows, C, act, dtype):
    o = ops()
    x = activations(rows, C, dtype, 1)
    dy = activations(rows, C, dtype, 2)
    a8 = o.act_quant8(x.to(DEV))
    h, d = act64(o.act_dequant8(a8, torch.float32).cpu().double(), act)
    half = torch.finfo(dtype).eps / 2
    got = o.act_dequant8(a8, act=act).cpu().double()
    assert ((got - h).abs() <= h.abs() * half + 1e-5 * h.abs().clamp(min=1.0)).all()
    got = o.act_bwd8(dy.to(DEV), a8, act).cpu().double()
    want = dy.double() * d
    assert ((got - want).abs() <= want.abs() * half + 1e-5 * dy.double().abs()).all()
    inplace = dy.to(DEV)
    assert o.act_bwd8(inplace, a8, act, out=inplace) is inplace and torch.equal(inplace.cpu().double(), got)
    # the transposed reader: the same values bit for bit, zero columns behind them
    for a in (0, act):
        t = o.act_dequant8_t(a8, act=a)
        assert t.shape[0] == C and t.shape[1] >= rows and t.shape[1] % 8 == 0
        assert torch.equal(t[:, :rows], o.act_dequant8(a8, act=a).t()) and (t[:, rows:] == 0).all()


def test_derivative_is_finite_far_out_and_nan_stays():
    o = ops()
    x = torch.zeros(1, 96)
    x[0, :32] = torch.linspace(-3e38, 3e38, 32)
    x[0, 32:64] = float("nan")
    x[0, 64:] = torch.linspace(-60, 60, 32)
    a8 = o.act_quant8(x.to(DEV))
    for act in (1, 2, 3):
        d = o.act_bwd8(torch.ones(1, 96, device=DEV), a8, act).cpu()
        v = o.act_dequant8(a8).cpu()
        assert torch.isnan(d[0, 32:64]).all()
        for sl in (slice(0, 32), slice(64, 96)):
            far = v[0, sl].abs() > 32
            # gelu' is 0 or 1 there; silu'(x) = s (1 + x (1 - s)), s < e^x, so |silu'(x)| < |x| e^x <= 32 e^-32 < 4.1e-13 for x <= -32
            assert ((d[0, sl][far] - (v[0, sl][far] > 0).float()).abs() <= (4.1e-13 if act == 1 else 0.0)).all()


def test_no_rows_streams_and_graph_replay():
    o = ops()
    a8 = o.act_quant8(torch.empty(0, 64, device=DEV))
    assert a8.rows == 0 and o.act_dequant8(a8).shape == (0, 64) and o.act_bwd8(torch.empty(0, 64, device=DEV), a8, 2).shape == (0, 64)
    with pytest.raises(ValueError):
        o.act_dequant8_t(a8)
    x = activations(300, 1000, torch.bfloat16).to(DEV)
    want = o.act_dequant8_t(o.act_quant8(x), act=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = o.act_dequant8_t(o.act_quant8(x), act=2)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    xs = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = o.act_quant8(xs)
        t, d = o.act_dequant8_t(kept, act=2), o.act_bwd8(xs, kept, 2)
    for i in range(3):
        xi = activations(300, 1000, torch.bfloat16, 10 + i).to(DEV)
        xs.copy_(xi)
        g.replay()
        k = o.act_quant8(xi)
        torch.cuda.synchronize()
        assert torch.equal(t, o.act_dequant8_t(k, act=2)) and torch.equal(d, o.act_bwd8(xi, k, 2))


def test_refusals():
    o = ops()
    x = torch.randn(8, 64, device=DEV)
    a8 = o.act_quant8(x)
    with pytest.raises(TypeError):
        o.act_quant8(x.half())
    with pytest.raises(ValueError):
        o.act_quant8(x.t()[:, ::2])
    with pytest.raises(ValueError):
        o.act_quant8(x, out=o.act_quant8(x[:4]))
    with pytest.raises(ValueError):
        o.act_bwd8(x[:4], a8, 2)
    with pytest.raises(o._lib.More4DHipError):
        o.act_bwd8(x, a8, 0)
    with pytest.raises(o._lib.More4DHipError):
        o.act_dequant8(a8, act=4)
    with pytest.raises(ValueError):
        o.act_dequant8(a8, out=torch.empty(8, 32, device=DEV))


# ------------------------------------------------------------------ the DiT block's stored activations
def _tiny(dtype):
    from more4d_amd.models import WanTransformer4DModel
    from test_dit_gpu import TINY
    from util import load_keys, load_npz
    from weights import fill
    z = load_npz("dit_tiny.npz")
    m = WanTransformer4DModel(**TINY)
    m.load_state_dict(fill(load_keys("dit_tiny_keys.json"), 1234))
    m = m.to(DEV, dtype).train()
    kw = dict(x=z["x"].to(DEV), t=z["t"].to(DEV), context=[z["ctx0"].to(DEV), z["ctx1"].to(DEV)], seq_len=int(z["seq_len_pad"]),
              clip_fea=z["clip"].to(DEV), y=z["y"].to(DEV), full_ref=z["full_ref"].to(DEV))
    return m, kw


def _grads(m, kw):
    m.zero_grad(set_to_none=True)
    pred = m(**kw)
    g = torch.Generator(device=DEV).manual_seed(7)
    (pred.float() * torch.randn(pred.shape, generator=g, device=DEV)).sum().backward()
    return pred.detach().clone(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_gradients_from_codes_equal_those_of_the_values_they_stand_for(dtype, monkeypatch):
    """The backward over a stash of codes against the same backward over a stash of plain tensors holding the codes' values.  All readers but
    two expand the codes to exactly those tensors; the two that read codes directly (act_dequant8_t, act_bwd8) evaluate GELU and its
    derivative in float32 like the plain kernels, in another order of operations: within one rounding to the type, eps / 2 relative, of each
    element of h^T and of the pre-activation's gradient (plus 1e-5 of their size, the float32 bound at the top of this file).  The last block's
    feed-forward gradients are linear in those two, and its incoming gradient is the same in both runs: eps of their rms.
    Behind the feed-forward the difference passes softmaxes, whose gradients are sums that cancel (the keys' dS sum to zero), so it can grow
    relative to what is left of them.  Both runs evaluate one formula on the same values: in float32 each is within 1e-3 of the exact gradient
    (the bound of the comparisons with the reference's gradients in test_train_gpu.py), so 2e-3 of each other; in bfloat16 the bound of the
    next test applies."""
    from more4d_amd import autograd, ops
    m, kw = _tiny(dtype)
    m.activation_budget_gb, m.activation_bits = 1e6, 8
    pred, coded = _grads(m, kw)
    assert m.last_full_blocks == len(m.blocks)
    monkeypatch.setattr(autograd.ops, "act_quant8", lambda t: ops.act_dequant8(_quant8(t)))
    pred2, plain = _grads(m, kw)
    assert torch.equal(pred, pred2) and coded.keys() == plain.keys()
    eps = max(torch.finfo(dtype).eps, 1e-5)
    direct = [f"blocks.{len(m.blocks) - 1}.ffn.{k}.{w}" for k in (0, 2) for w in ("weight", "bias")]
    assert set(direct) <= coded.keys()
    for n in coded:
        a, b = coded[n].double(), plain[n].double()
        tol = eps if n in direct else 2e-3 if dtype == torch.float32 else 0.05
        assert float((a - b).norm()) <= tol * float(b.norm()) + 1e-9, (n, float((a - b).norm() / b.norm()))


from more4d_amd.ops import act_quant8 as _quant8  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("full", [True, False])
def test_model_with_8_bit_activations(dtype, full):
    """activation_bits = 8: the same prediction bit for bit; gradients near those of stored tensors; more blocks in the same budget.  A code is off
    by at most half a step of max / 64 of its block, for normal data a uniform error of rms below (2.5 / 64) / sqrt(12) = 1.2 % of the block's
    rms; at most eight rounded tensors enter a gradient: sqrt(8) * 1.2 % = 3.4 %, asked for: 5 %.  That is relative to the terms of a gradient's
    sum.  The key projections (biases, norm weights, and weights for the part of their inputs that all keys share) sum dS over the keys, which for
    a softmax sums to zero: what the RMSNorm leaves is the spread of the keys' 1 / rms, 1 / sqrt(2 * 128) = 1 / 16 of the terms at 128 channels, so for them the same error is up to 16 times 3.4 % of the
    result: 54 %."""
    m, kw = _tiny(dtype)
    C, F = m.dim, m.ffn_dim
    m.activation_budget_gb = 1e6
    if not full:
        B, _, f, h, w = kw["x"].shape
        rows = B * (-(-(f + 1) * (h // 2) * (w // 2) // 8) * 8)      # tokens and the reference frame's
        es = 4 if dtype == torch.float32 else 2
        m.activation_budget_gb = (rows * (2 * C * es + m.num_heads * 4) * len(m.blocks) + rows * (6 * C + F) * es * 0.6) / 2 ** 30
    ref = _grads(m, kw)
    blocks16 = m.last_full_blocks
    m.activation_bits = 8
    got = _grads(m, kw)
    assert torch.equal(ref[0], got[0])
    assert m.last_full_blocks > blocks16 if not full else m.last_full_blocks == blocks16 == len(m.blocks)
    for n, b in ref[1].items():
        a, b = got[1][n].double(), b.double()
        tol = 0.54 if ".k." in n or ".k_img." in n or ".norm_k" in n else 0.05
        assert float((a - b).norm()) <= tol * float(b.norm()) + 1e-9, (n, float((a - b).norm() / b.norm()))
    m.activation_bits = 4
    with pytest.raises(ValueError):
        m(**kw)
