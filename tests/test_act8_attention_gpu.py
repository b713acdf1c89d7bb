"""activation_bits = 8 and the self-attention's backward.  P = exp(S - lse) and delta = rowsum(dO o) are a softmax's gradient only if lse and o are
those of the q, k, v at hand: then every row of P sums to 1 and every row of dS to 0."""
import pytest
import torch

from test_act8_gpu import _grads, _tiny

pytestmark = pytest.mark.gpu


def _large_logits(m):
    """uneven norm weights and scores of standard deviation around 4 in the self-attention, as trained models have them"""
    g = torch.Generator().manual_seed(11)
    with torch.no_grad():
        for blk in m.blocks:
            for n, s in ((blk.self_attn.norm_q, 3.0), (blk.self_attn.norm_k, 1.0)):
                n.weight.mul_((s * torch.exp(0.5 * torch.randn(n.weight.shape, generator=g))).to(n.weight))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("store", [1, 2, 3])
def test_the_self_attention_backward_gets_what_belongs_together(dtype, store, monkeypatch):
    """Every call's lse (to the base 2) and o against float64 on the q, k, v of the same call.  lse: scores to 2^-23 of a sum of head_dim terms (float32), in bfloat16
    probabilities rounded to the type before they are summed, at most 2^-8 of the sum.  o: probabilities and result rounded to the type, two halves of eps
    (float32: 1e-4, accumulations included)."""
    from more4d_amd import autograd, ops
    m, kw = _tiny(dtype)
    _large_logits(m)
    m.activation_budget_gb, m.activation_bits = 1e6, 8
    forward = autograd.BlockFn.apply    # every block in this tier
    monkeypatch.setattr(autograd.BlockFn, "apply", staticmethod(lambda *a: forward(*a[:9], (store, 8), *a[10:])))
    seen, real = [], ops.attention_bwd

    def spy(q, k, v, o, d_o, lse, *, B, Lq, Lk, Lk_rows, heads, head_dim, scale=None, **kws):
        def split(t, L):
            return t.double().view(B, L, heads, head_dim).transpose(1, 2)
        s = split(q, Lq) @ split(k, Lk_rows)[:, :, :Lk].transpose(2, 3).contiguous() * (head_dim ** -0.5 if scale is None else scale)
        want = torch.softmax(s, -1) @ split(v, Lk_rows)[:, :, :Lk].contiguous()
        half = torch.finfo(dtype).eps / 2
        off = (lse.view(B, heads, Lq).double() - torch.logsumexp(s, -1) * 1.4426950408889634).abs().max()
        err = (split(o, Lq) - want).norm() / want.norm()
        seen.append((Lq == Lk_rows, float(off), float(err), float(s.std())))
        return real(q, k, v, o, d_o, lse, B=B, Lq=Lq, Lk=Lk, Lk_rows=Lk_rows, heads=heads, head_dim=head_dim, scale=scale, **kws)

    monkeypatch.setattr(ops, "attention_bwd", spy)
    _grads(m, kw)
    mine = [t for t in seen if t[0]]
    assert len(mine) == len(m.blocks) and max(t[3] for t in mine) > 2
    for _, off, err, _ in seen:
        assert off <= (1e-4 if dtype == torch.float32 else 2.0 ** -8) and err <= (1e-4 if dtype == torch.float32 else 2.0 ** -7), seen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_at_large_logits(dtype):
    """Gradients against those of stored tensors.  The self-attention's backward is linear in dO and works on exact q, k, v, lse and o, and a softmax's
    dS sums to zero for every dO: what the rounded tensors behind it (rms 1.2 % each, at most six: 3 %) put on dO passes it at its own size, key
    projections included.  The cross-attention's queries are rounded: its scores, of standard deviation around 1, move by 1.2 % of their size, P
    likewise.  sqrt(3^2 + 1.2^2) = 3.2 %, asked for: 8 %, of every gradient.
    In bfloat16 the image keys' biases are sums that cancel to the size of the type's own roundings, in the run that stores tensors too: how far that run
    is from the float32 model of the same weights is added, twice for the two runs."""
    m, kw = _tiny(dtype)
    _large_logits(m)
    m.activation_budget_gb = 1e6
    ref = _grads(m, kw)
    m.activation_bits = 8
    got = _grads(m, kw)
    own = dict.fromkeys(ref[1], 0.0)
    if dtype != torch.float32:
        m.activation_bits = 16
        exact = _grads(m.float(), kw)[1]
        own = {n: float((b.double() - exact[n].double()).norm() / (exact[n].double().norm() + 1e-12)) for n, b in ref[1].items()}
    assert torch.equal(ref[0], got[0])
    off = {n: float((got[1][n].double() - b.double()).norm() / (b.double().norm() + 1e-12)) for n, b in ref[1].items()}
    bad = {n: (v, own[n]) for n, v in off.items() if v > 0.08 + 2 * own[n]}
    assert not bad, bad


@pytest.mark.parametrize("bits", [8, 16])
def test_the_backward_lets_go_of_what_it_has_used(bits, monkeypatch):
    """By the time a block's backward has come to its self-attention, the codes of that block are gone, and with 16 bits the tensors of its feed-forward."""
    import weakref
    from more4d_amd import autograd, ops
    m, kw = _tiny(torch.bfloat16)
    m.activation_budget_gb, m.activation_bits = 1e6, bits
    kept, alive, real, quant = [], [], ops.attention_bwd, ops.act_quant8
    forward = autograd.block_backward

    def forward_half(*a, **k):
        out = forward(*a, **k)
        if k.get("forward_only") and bits == 16:
            kept.append([weakref.ref(out[1][n]) for n in ("pre", "y2")])
        elif k.get("forward_only"):
            kept.append([])
        return out

    def quantized(t):
        a8 = quant(t)
        kept[-1].append(weakref.ref(a8.buf))
        return a8

    def spy(q, k, *a, Lq, Lk_rows, **kws):
        if Lq == Lk_rows:
            alive.append(sum(r() is not None for r in kept.pop()))
        return real(q, k, *a, Lq=Lq, Lk_rows=Lk_rows, **kws)

    monkeypatch.setattr(autograd, "block_backward", forward_half)
    monkeypatch.setattr(ops, "act_quant8", quantized)
    monkeypatch.setattr(ops, "attention_bwd", spy)
    _grads(m, kw)
    assert len(alive) == len(m.blocks) and not any(alive), alive
