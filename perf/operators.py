"""Cases, plain forms and calls of two groups of operators.

Low-rank adapters beside a shared projection.  x [M, K] holds the rows of several requests one behind the other; request j owns
lengths[j] rows and names an adapter g (or -1: none).  With W [N, K] shared and (A_g [r, K], B_g [N, r], s_g) of each adapter

    y = x W^T + bias + s_g (x A_g^T) B_g^T                                        ("serve": the forward pass)
    dx = dy W + s_g (dy B_g) A_g,   dA_g = s_g sum_rows (dy B_g)^T x8,   dB_g = s_g sum_rows dy^T (x A_g^T)
                                                                                  ("train": forward and backward, W and bias frozen)

where x8 is the input that the forward kept for the backward: x itself, or its 8-bit form.

Activations kept in 8 bits.  Each row is cut into blocks of 32 consecutive channels (the last one may be shorter); a block has one
power of two 2^e, e the smallest integer >= -126 with max|x| <= 127 * 2^e (at most 121; beyond it the codes saturate), and the codes
round_half_even(x / 2^e) in [-127, 127].  A block that holds an infinity or NaN stands for NaN throughout.

    "store":  the values that the codes of x stand for                            (written by the forward, read back by the backward)
    "ffn":    keep `pre`, then in the backward  dpre = dh * act'(pre8)  and  h^T = act(pre8)^T, the operand of the weight gradient
"""
import math
import random  # noqa: F401  (the type of draw's argument)

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ACTS = {"silu": 1, "gelu_tanh": 2, "gelu_erf": 3}      # the framework's activation codes
BLOCK = 32


def listed():
    return [
        # modulation vectors of two samples (a guidance pair of two requests), each with its own adapter: 1536 -> 6 x 1536
        {"name": "serve_mod_2rows", "op": "serve", "dtype": "bf16", "K": 1536, "N": 9216, "rank": 16, "lengths": "1,1", "ids": "1,0",
         "adapters": 2},
        # the same projection of the large model for eight requests, one of them without an adapter, two sharing one
        {"name": "serve_mod_8rows", "op": "serve", "dtype": "bf16", "K": 5120, "N": 30720, "rank": 32, "lengths": "1,1,1,1,1,1,1,1",
         "ids": "3,0,-1,4,1,0,2,5", "adapters": 6},
        # text embedding of prompts of different lengths, packed without padding; an empty prompt among them, odd rank
        {"name": "serve_text_ragged", "op": "serve", "dtype": "bf16", "K": 4096, "N": 5120, "rank": 12,
         "lengths": "512,77,1,0,226,131,39", "ids": "0,2,1,1,-1,2,3", "adapters": 4},
        # the parity type at the small model's width
        {"name": "serve_text_fp32", "op": "serve", "dtype": "fp32", "K": 4096, "N": 1536, "rank": 16, "lengths": "77,19,226",
         "ids": "1,-1,0", "adapters": 2},
        # video tokens of a guidance pair, one adapter for both halves: attention projection of the large model
        {"name": "serve_dit_proj", "op": "serve", "dtype": "bf16", "K": 5120, "N": 5120, "rank": 64, "lengths": "21840,21840",
         "ids": "0,0", "adapters": 1},
        # two videos of one batch with an adapter each, the wide projection of the feed-forward
        {"name": "serve_dit_ffn", "op": "serve", "dtype": "bf16", "K": 5120, "N": 13824, "rank": 128, "lengths": "21840,20280",
         "ids": "1,0", "adapters": 2},
        # training the small model's adapter on one short clip, odd row count, input kept in 8 bits
        {"name": "train_small_8bit", "op": "train", "dtype": "bf16", "K": 1536, "N": 1536, "rank": 16, "lengths": "1573", "ids": "0",
         "adapters": 1, "bits": 8},
        # training the large model's adapter on one full clip, input kept in 8 bits
        {"name": "train_dit_8bit", "op": "train", "dtype": "bf16", "K": 5120, "N": 5120, "rank": 64, "lengths": "21840", "ids": "0",
         "adapters": 1, "bits": 8},
        # several tasks trained side by side on clips of different lengths, input kept as it is
        {"name": "train_tasks_16bit", "op": "train", "dtype": "bf16", "K": 1536, "N": 8960, "rank": 32,
         "lengths": "1560,3120,780,4680,1,1560", "ids": "0,1,-1,2,3,0", "adapters": 4, "bits": 16},
        # an attention output kept for the backward, odd rows
        {"name": "store_small", "op": "store", "dtype": "bf16", "rows": 1573, "C": 1536},
        # the float32 residual stream at the width of the large model
        {"name": "store_fp32", "op": "store", "dtype": "fp32", "rows": 21840, "C": 5120},
        # the feed-forward's widest tensor, kept in 8 bits and used in the backward
        {"name": "ffn_dit", "op": "ffn", "dtype": "bf16", "rows": 21840, "C": 13824, "act": "gelu_tanh"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_requests(rng, rows):
    n = min(rows, _log_int(rng, 1, 24))
    cuts = sorted(rng.randint(0, rows) for _ in range(n - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    adapters = rng.randint(1, max(1, min(n, 12)))
    ids = [rng.randint(-1, adapters - 1) for _ in lengths]
    if max(ids) < 0:
        ids[lengths.index(max(lengths))] = 0
    return ",".join(map(str, lengths)), ",".join(map(str, ids)), adapters


def draw(rng):
    op = rng.choice(["serve", "serve", "serve", "train", "train", "store", "ffn"])
    if op in ("store", "ffn"):
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        C = rng.choice([_log_int(rng, 16, 1728) * 8, _log_int(rng, 64, 13824)])
        rows = min(_log_int(rng, 1, 24000), (3 * 10 ** 8 if dtype == "bf16" else 12 * 10 ** 7) // C)
        case = {"op": op, "dtype": dtype, "rows": rows, "C": C}
        if op == "ffn":
            case["act"] = rng.choice(sorted(ACTS))
        return case
    while True:
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        K, N = 8 * _log_int(rng, 32, 1728), 4 * _log_int(rng, 64, 7680)
        rows = _log_int(rng, 1, 43680)
        limit = (3e12 if op == "serve" else 1.4e12) if dtype == "bf16" else 1e11
        if 2.0 * rows * K * N > limit:
            continue
        lengths, ids, adapters = _draw_requests(rng, rows)
        case = {"op": op, "dtype": dtype, "K": K, "N": N, "rank": _log_int(rng, 2, 128), "lengths": lengths, "ids": ids,
                "adapters": adapters}
        if op == "train":
            case["bits"] = rng.choice([8, 16])
        if work(case)["bytes"] <= 3e9:
            return case


def _requests(case):
    lengths = [int(v) for v in case["lengths"].split(",")]
    ids = [int(v) for v in case["ids"].split(",")]
    return lengths, ids


def _activations(g, rows, C, dtype):
    """Activations as a transformer block has them: unit scale, a few channels several times larger."""
    ch = torch.exp(0.5 * torch.randn(C, generator=g, device="cuda"))
    ch[torch.rand(C, generator=g, device="cuda") < 0.01] *= 8.0
    return (torch.randn(rows, C, generator=g, device="cuda") * ch).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"op": case["op"], "own": own}
    if case["op"] in ("store", "ffn"):
        st["x"] = _activations(g, case["rows"], case["C"], dt)
        if case["op"] == "ffn":
            st["act"] = case["act"]
            st["dh"] = (0.01 * torch.randn(case["rows"], case["C"], generator=g, device="cuda")).to(dt)
        return st
    lengths, ids = _requests(case)
    K, N, r, G = case["K"], case["N"], case["rank"], case["adapters"]
    x = _activations(g, sum(lengths), K, dt)
    w = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).to(dt)
    bias = (0.1 * torch.randn(N, generator=g, device="cuda")).to(dt)
    a = (torch.randn(G, r, K, generator=g, device="cuda") * K ** -0.5).to(dt)
    b = (0.1 * torch.randn(G, N, r, generator=g, device="cuda")).to(dt)
    scale = [0.5 + 0.25 * (i % 5) for i in range(G)]
    st.update(x=x, w=w, bias=bias, a=a, b=b, scale=scale, lengths=lengths, ids=ids)
    if case["op"] == "train":
        st["bits"] = case["bits"]
        st["dy"] = (0.01 * torch.randn(sum(lengths), N, generator=g, device="cuda")).to(dt)
        for t in (x, a, b):
            t.requires_grad_(True)
    if own:
        from more4d_amd import ops
        st["plan"] = ops.AdapterPlan(lengths, ids, "cuda")
        st["scale_dev"] = torch.tensor(scale, device="cuda")
        if case["op"] == "serve":
            st["bank"] = ops.AdapterBank(a, b, scale)
    return st


# ------------------------------------------------------------------ plain forms
def _spans(lengths, ids):
    pos = 0
    for n, i in zip(lengths, ids):
        if n > 0 and i >= 0:
            yield slice(pos, pos + n), i
        pos += n


def _plain_codes(x):
    """float32 [rows, C] -> the values that its 8-bit codes stand for."""
    rows, C = x.shape
    xb = torch.nn.functional.pad(x, (0, -C % BLOCK)).view(rows, -1, BLOCK)
    top = xb.abs().amax(dim=-1, keepdim=True)
    m, ex = torch.frexp(top)
    e = (ex - torch.where(m <= 127.0 / 128.0, 7, 6)).clamp(-126, 121)
    val = torch.ldexp(torch.round(torch.ldexp(xb, -e)).clamp(-127, 127), e)
    val = torch.where(torch.isfinite(xb).all(dim=-1, keepdim=True), val, torch.full_like(val, float("nan")))
    return val.view(rows, -1)[:, :C]


def _plain_act(x, act):
    """(act(x), act'(x))"""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return x * s, s * (1.0 + x * (1.0 - s))
    if act == "gelu_erf":
        c = 0.5 * (1.0 + torch.erf(x * 0.5 ** 0.5))
        return x * c, c + x * torch.exp(-0.5 * x * x) * (2.0 * math.pi) ** -0.5
    k, q = (2.0 / math.pi) ** 0.5, 0.044715
    t = torch.tanh(k * (x + q * x * x * x))
    return 0.5 * x * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * k * (1.0 + 3.0 * q * x * x)


def _plain_forward(st):
    x = st["x"].detach().float()
    y = x @ st["w"].float().t() + st["bias"].float()
    for rows, i in _spans(st["lengths"], st["ids"]):
        y[rows] += st["scale"][i] * ((x[rows] @ st["a"][i].detach().float().t()) @ st["b"][i].detach().float().t())
    return y.to(st["x"].dtype)


def _plain_train(st):
    y = _plain_forward(st)
    dt = y.dtype
    x, dy = st["x"].detach().float(), st["dy"].float()
    a, b = st["a"].detach().float(), st["b"].detach().float()
    x8 = _plain_codes(x) if st["bits"] == 8 else x
    dx = dy @ st["w"].float()
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for rows, i in _spans(st["lengths"], st["ids"]):
        v = st["scale"][i] * (dy[rows] @ b[i])
        dx[rows] += v @ a[i]
        da[i] += v.t() @ x8[rows]
        db[i] += dy[rows].t() @ (st["scale"][i] * (x[rows] @ a[i].t()))
    return y, dx.to(dt), da.to(dt), db.to(dt)


def _run_plain(st):
    if st["op"] == "serve":
        return _plain_forward(st)
    if st["op"] == "train":
        return _plain_train(st)
    dt = st["x"].dtype
    val = _plain_codes(st["x"].float())
    if st["op"] == "store":
        return val.to(dt)
    h, dact = _plain_act(val, st["act"])
    return (st["dh"].float() * dact).to(dt), h.t().contiguous().to(dt)


# ------------------------------------------------------------------ the framework's operators
def _run_own(st):
    from more4d_amd import autograd, ops
    if st["op"] == "serve":
        return ops.linear_adapters(st["x"], st["w"], st["bias"], st["bank"], st["plan"])
    if st["op"] == "train":
        y = autograd.AdapterLinearFn.apply(st["x"], st["w"], st["bias"], st["a"], st["b"], st["scale_dev"], st["plan"], st["bits"])
        return (y.detach(),) + torch.autograd.grad(y, (st["x"], st["a"], st["b"]), st["dy"])
    kept = ops.act_quant8(st["x"])
    if st["op"] == "store":
        return ops.act_dequant8(kept)
    act = ACTS[st["act"]]
    return ops.act_bwd8(st["dh"], kept, act), ops.act_dequant8_t(kept, act=act)[:, :st["x"].shape[0]]


def run(state):
    return _run_own(state) if state["own"] else _run_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("store", "ffn"):
        n = case["rows"] * case["C"]
        code = n + case["rows"] * -(-case["C"] // BLOCK)      # a byte per code and one per block, written once and read once
        if case["op"] == "store":
            return {"bytes": 2 * n * es + 2 * code, "flops": 4 * n}
        return {"bytes": 4 * n * es + 2 * code, "flops": 40 * n}
    lengths, ids = _requests(case)
    M, K, N, r = sum(lengths), case["K"], case["N"], case["rank"]
    on = sum(n for n, i in zip(lengths, ids) if i >= 0)
    used = len({i for n, i in zip(lengths, ids) if i >= 0 and n > 0})
    ad = used * r * (K + N)
    if case["op"] == "serve":
        return {"bytes": es * (M * K + N * K + N + ad + M * N), "flops": 2 * M * K * N + 2 * on * r * (K + N)}
    # x and dy in, the weights, y and dx out; the kept 8-bit input is written once and read once
    kept = 2 * (M * K + M * -(-K // BLOCK)) if case["bits"] == 8 else 0
    return {"bytes": es * (2 * M * K + 2 * M * N + N * K + N + 2 * ad) + kept, "flops": 4 * M * K * N + 6 * on * r * (K + N)}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_codes(x):
    """Codes by search over the powers of two, block by block, in 64 bits."""
    rows, C = x.shape
    nb = -(-C // BLOCK)
    out = torch.empty_like(x)
    for j in range(nb):
        blk = x[:, j * BLOCK:(j + 1) * BLOCK]
        top = blk.abs().max(dim=1, keepdim=True).values
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -160))) - 8
        for _ in range(4):
            e = torch.where(127.0 * torch.exp2(e) < top, e + 1, e)
        e = e.clamp(-126, 121)
        step = torch.exp2(e)
        out[:, j * BLOCK:(j + 1) * BLOCK] = (blk / step).round().clamp(-127, 127) * step
    return out


def _exact_act(x, act):
    x = x.clone().requires_grad_(True)
    if act == "silu":
        h = x * torch.sigmoid(x)
    elif act == "gelu_erf":
        h = 0.5 * x * torch.erfc(-x / math.sqrt(2.0))
    else:
        h = x * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3))
    (d,) = torch.autograd.grad(h.sum(), x)
    return h.detach(), d


def exact(case, seed):
    was = globals()["own"]
    globals()["own"] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()["own"] = was
    x = st["x"].detach().double()
    if case["op"] == "store":
        return _exact_codes(x)
    if case["op"] == "ffn":
        h, d = _exact_act(_exact_codes(x), case["act"])
        return st["dh"].double() * d, h.t().contiguous()
    lengths, ids = _requests(case)
    row_id = torch.from_numpy(np.repeat(np.array(ids), np.array(lengths))).cuda()
    w, bias = st["w"].double(), st["bias"].double()
    a, b = st["a"].detach().double(), st["b"].detach().double()
    train = case["op"] == "train"
    y = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    if train:
        dy = st["dy"].double()
        x8 = _exact_codes(x) if case["bits"] == 8 else x
        dx, da, db = torch.empty_like(x), torch.zeros_like(a), torch.zeros_like(b)
    # one merged weight per adapter, applied to the rows that name it
    for i in range(-1, case["adapters"]):
        rows = torch.nonzero(row_id == i).flatten()
        if rows.numel() == 0:
            continue
        merged = w if i < 0 else w + st["scale"][i] * (b[i] @ a[i])
        y[rows] = x[rows] @ merged.t() + bias
        if train:
            dx[rows] = dy[rows] @ merged
            if i >= 0:
                da[i] = st["scale"][i] * (b[i].t() @ (dy[rows].t() @ x8[rows]))
                db[i] = st["scale"][i] * ((dy[rows].t() @ x[rows]) @ a[i].t())
    return (y, dx, da, db) if train else y
