"""Cases of the 8-bit integer operators (W8A8: int8 weights with a scale for each output channel, int8 activations with a scale
for each token) and of the whole MoE layer for a few tokens.

What a program with the MoE block has them do: quantise rows; one linear layer (the attention projections of a quantised
model); the expert products of a prefill, fed through the routing's permutation; and, while a few sequences are being decoded,
the whole layer (router, top-k, experts, weighted sum) on bf16, fp16, int4 (W4A16) or int8 experts.

Sizes are those of the repository's configurations and tests: the Qwen3-30B-A3B layer (hidden 2048, 128 experts, 8 per token,
expert width 768), smaller layers with it, the attention-shape linears, and batches from one row on.
"""
import os
import sys

import torch

own = False

GROUP = 128
QWEN = {"H": 2048, "E": 128, "K": 8, "I": 768}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # rows of a prompt of odd length in front of a projection, the last ones padding (all zero)
        {"name": "quantize_777", "kind": "quantize", "rows": 777, "cols": 2048, "padding": 9, "dtype": "bf16"},
        # the expert activations of 4096 tokens, 8 experts each, in front of the down projection
        {"name": "quantize_32768", "kind": "quantize", "rows": 32768, "cols": 768, "padding": 0, "dtype": "bf16"},
        # an attention projection while one sequence is decoded: the smallest call
        {"name": "linear_1", "kind": "linear", "M": 1, "Kd": 2048, "N": 4096, "dtype": "bf16"},
        # the output projection of a prompt of odd length, in fp16
        {"name": "linear_500", "kind": "linear", "M": 500, "Kd": 4096, "N": 2048, "dtype": "fp16"},
        # a projection of 4096 tokens
        {"name": "linear_4096", "kind": "linear", "M": 4096, "Kd": 2048, "N": 4096, "dtype": "bf16"},
        # gate and up projections with SwiGLU of a small batch whose rows are grouped by expert, some experts without any
        {"name": "experts_swiglu_96", "kind": "swiglu", "T": 96, "gather": True, "skew": 1.2, "dtype": "bf16", **QWEN},
        # the same for 4096 tokens: the largest case
        {"name": "experts_swiglu_4096", "kind": "swiglu", "T": 4096, "gather": True, "skew": 0.0, "dtype": "bf16", **QWEN},
        # the down projection behind it for a prompt of odd length
        {"name": "experts_down_777", "kind": "down", "T": 777, "skew": 0.0, "dtype": "bf16", **QWEN},
        # one sequence being decoded: the whole layer with bf16 experts
        {"name": "layer_bf16_1", "kind": "layer", "experts": "dense", "T": 1, "residual": False, "dtype": "bf16", **QWEN},
        # 13 sequences on int4 experts, the decoder layer's residual with it
        {"name": "layer_w4_13", "kind": "layer", "experts": "w4", "T": 13, "residual": True, "dtype": "bf16", **QWEN},
        # five sequences on int8 experts
        {"name": "layer_w8_5", "kind": "layer", "experts": "w8", "T": 5, "residual": False, "dtype": "bf16", **QWEN},
        # the largest batch of the layer call, fp16 experts
        {"name": "layer_fp16_16", "kind": "layer", "experts": "dense", "T": 16, "residual": False, "dtype": "fp16", **QWEN},
    ]


def _log_int(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _layer_shape(rng):
    """The Qwen3-30B-A3B layer, or one no larger of the same family."""
    if rng.random() < 0.5:
        return dict(QWEN)
    E = rng.choice([8, 16, 32, 64, 128])
    return {"H": 128 * rng.randint(2, 16), "E": E, "K": rng.choice([1, 2, 4, 6, 8]), "I": 128 * rng.randint(1, 6)}


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "swiglu", "down", "layer", "layer", "layer"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "quantize":
        cols = _log_int(rng, 16, 8192) if rng.random() < 0.4 else 64 * rng.randint(2, 64)
        return {"kind": kind, "rows": _log_int(rng, 1, 32768 if cols <= 2048 else 4096), "cols": cols,
                "padding": rng.choice([0, 0, 1]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "linear":
        c = {"kind": kind, "M": _log_int(rng, 1, 4096), "Kd": 16 * rng.randint(8, 256), "N": 16 * rng.randint(16, 256),
             "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if rng.random() < 0.2:       # sizes off every grid
            c.update(M=min(c["M"], 512), Kd=rng.randint(33, 1500), N=rng.randint(9, 1500))
        return c
    shape = _layer_shape(rng)
    if kind == "layer":
        experts = rng.choice(["dense", "w4", "w8"])
        return {"kind": kind, "experts": experts, "T": _log_int(rng, 1, 16), "residual": rng.random() < 0.5,
                "dtype": "bf16" if experts == "w4" else half, **shape}
    c = {"kind": kind, "T": _log_int(rng, 1, 4096), "skew": rng.choice([0.0, 0.0, 1.2]), "dtype": half, **shape}
    if kind == "swiglu":
        c["gather"] = rng.random() < 0.7
    return c


# ---- inputs ---------------------------------------------------------------------------------------------
def _normal(gen, shape, std, dtype):
    return torch.empty(shape, dtype=dtype, device=gen.device).normal_(0.0, std, generator=gen)


def _hidden(gen, shape, dtype):
    """Hidden states: about N(0, 1), with a few channels that are an order of magnitude larger in every row."""
    big = 1.0 + 9.0 * (torch.rand(shape[-1], generator=gen, device=gen.device) < 0.01).to(dtype)
    return _normal(gen, shape, 1.0, dtype) * big


def _int8(gen, lead, n, kd):
    """int8 weights [*lead, n, kd], bell-shaped over the whole range, and a scale for each row such that a weight is about
    N(0, 0.02)."""
    q = torch.empty((*lead, n, kd), dtype=torch.float16, device=gen.device).normal_(0.0, 32.0, generator=gen)
    q = q.round_().clamp_(-127, 127).to(torch.int8)
    scales = (torch.rand((*lead, n), generator=gen, device=gen.device) * 0.4 + 0.8) * (0.02 / 32)
    return q, scales


def _bits(gen, shape):
    return torch.randint(-2 ** 31, 2 ** 31 - 1, shape, generator=gen, device=gen.device, dtype=torch.int32)


def _int4(gen, lead, kd, n):
    """Packed int4 weights as a quantised checkpoint holds them: bell-shaped around the zero point (the sum of two uniform 0..7
    and one bit), zero points 7 or 8, scales such that a weight is about N(0, 0.02)."""
    qw = (_bits(gen, (*lead, kd // 8, n)) & 0x77777777) + (_bits(gen, (*lead, kd // 8, n)) & 0x77777777)
    qw = qw + (_bits(gen, (*lead, kd // 8, n)) & 0x11111111)
    scales = (torch.rand(*lead, kd // GROUP, n, generator=gen, device=gen.device) * 0.003 + 0.0045).to(torch.bfloat16)
    qz = (_bits(gen, (*lead, kd // GROUP, n // 8)) & 0x11111111) + 0x77777777
    return qw, scales, qz


def _routing(gen, c):
    """K different experts for each of T tokens (with skew s, expert r is r ** -s as popular as the first), as the permutation
    of the slots by expert and its offsets."""
    T, E, K = c["T"], c["E"], c["K"]
    score = torch.rand(T, E, generator=gen, device=gen.device).log().neg().log().neg()        # Gumbel noise
    score = score - c["skew"] * torch.arange(1, E + 1, device=gen.device).float().log()
    ids = score.topk(K, dim=1).indices.reshape(-1)
    perm = torch.sort(ids, stable=True).indices.to(torch.int32)
    counts = torch.bincount(ids, minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=gen.device)
    offsets[1:] = counts.cumsum(0)
    return perm, offsets


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = c["kind"], DTYPES[c["dtype"]]
    s = {"kind": kind, "dtype": dtype}
    if kind == "quantize":
        s["x"] = _hidden(gen, (c["rows"], c["cols"]), dtype)
        s["x"][c["rows"] - min(c["padding"], c["rows"]):] = 0
        return s
    if kind == "linear":
        s["x"] = _hidden(gen, (c["M"], c["Kd"]), dtype)
        s["w"], s["scales"] = _int8(gen, (), c["N"], c["Kd"])
        return s
    H, E, K, I, T = c["H"], c["E"], c["K"], c["I"], c["T"]
    if kind in ("swiglu", "down"):
        s["perm"], s["offsets"] = _routing(gen, c)
        s["bounds"] = s["offsets"].tolist()          # the plain form goes expert by expert
        s["top_k"] = K
        if kind == "swiglu":
            s["gather"] = c["gather"]
            s["x"] = _hidden(gen, (T, H), dtype)
            if not c["gather"]:
                s["x"] = s["x"][s["perm"].long() // K]
            s["w"], s["scales"] = _int8(gen, (E,), 2 * I, H)
        else:
            s["x"] = _normal(gen, (T * K, I), 0.5, dtype) * _normal(gen, (T * K, I), 0.5, dtype)
            s["w"], s["scales"] = _int8(gen, (E,), H, I)
        return s
    s["experts"], s["top_k"], s["inter"] = c["experts"], K, I
    s["x"] = _hidden(gen, (T, H), dtype)
    s["residual"] = _normal(gen, (T, H), 1.0, dtype) if c["residual"] else None
    s["router"] = _normal(gen, (E, H), 0.02, dtype)
    if c["experts"] == "dense":
        s["gate_up"], s["down"] = _normal(gen, (E, 2 * I, H), 0.02, dtype), _normal(gen, (E, H, I), 0.02, dtype)
    elif c["experts"] == "w8":
        s["gate_up"], s["gate_up_scales"] = _int8(gen, (E,), 2 * I, H)
        s["down"], s["down_scales"] = _int8(gen, (E,), H, I)
    else:
        s["gate"], s["up"], s["down"] = _int4(gen, (E,), H, I), _int4(gen, (E,), H, I), _int4(gen, (E,), I, H)
    return s


# ---- the plain form -------------------------------------------------------------------------------------
def _plain_quantize(x):
    """Symmetric int8 rows: scale = max|x| / 127 as an fp32 number, q = the whole number next to x / scale, halves to even (in 64
    bits: the quotient may lie beside a half).  A row of zeros has scale 0."""
    v = x.double()
    scale = (v.abs().amax(dim=-1) / 127.0).float()
    step = scale.double().unsqueeze(-1)
    q = torch.where(step > 0, v / torch.where(step > 0, step, 1.0), 0.0).round().clamp(-127, 127)
    return q, scale


def _plain_matmul(q, w):
    """Sums of products of whole numbers pass 2^24, so in 64 bits; then 32 for the scales."""
    return (q.double() @ w.double().mT).float()


def _plain_silu(g):
    return g / (1.0 + torch.exp(-g))


def _plain_unpack(qw, scales, qz):
    """[n, K/8, N] words -> fp32 weights [n, N, K]."""
    nib = 4 * torch.arange(8, device=qw.device, dtype=torch.int32)
    q = ((qw.unsqueeze(2) >> nib.view(1, 1, 8, 1)) & 15).flatten(1, 2)
    z = ((qz.unsqueeze(3) >> nib) & 15).flatten(2, 3)
    w = (q.float().unflatten(1, (-1, GROUP)) - z.float().unsqueeze(2)) * scales.float().unsqueeze(2)
    return w.flatten(1, 2).mT


def _plain_layer(s):
    x, K, T = s["x"], s["top_k"], s["x"].shape[0]
    logits = x.double() @ s["router"].double().mT
    top, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    weights = torch.softmax(top, dim=-1)[:, :K]
    weights = (weights / weights.sum(dim=-1, keepdim=True)).float()
    ids = ids[:, :K].reshape(-1)
    if s["experts"] == "w8":
        q, sx = (t.repeat_interleave(K, dim=0) for t in _plain_quantize(x))
        gu = _plain_matmul(q.unsqueeze(1), s["gate_up"][ids]).squeeze(1) * sx.unsqueeze(1) * s["gate_up_scales"][ids]
        h = _plain_silu(gu[:, :s["inter"]]) * gu[:, s["inter"]:]
        q, sh = _plain_quantize(h)
        y = _plain_matmul(q.unsqueeze(1), s["down"][ids]).squeeze(1) * sh.unsqueeze(1) * s["down_scales"][ids]
    else:
        rows = x.float().repeat_interleave(K, dim=0).unsqueeze(2)
        if s["experts"] == "dense":
            gu = (s["gate_up"][ids].float() @ rows).squeeze(2)
            g, u = gu[:, :s["inter"]], gu[:, s["inter"]:]
            wd = s["down"][ids].float()
        else:
            g, u = ((_plain_unpack(*(t[ids] for t in s[p])) @ rows).squeeze(2) for p in ("gate", "up"))
            wd = _plain_unpack(*(t[ids] for t in s["down"]))
        y = (wd @ (_plain_silu(g) * u).unsqueeze(2)).squeeze(2)
    y = (y.view(T, K, -1) * weights.unsqueeze(2)).sum(dim=1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["dtype"])


def _plain(s):
    kind = s["kind"]
    if kind == "quantize":
        q, scale = _plain_quantize(s["x"])
        return {"q": q.to(torch.int8), "scale": scale}
    if kind == "layer":
        return _plain_layer(s)
    q, sx = _plain_quantize(s["x"])
    if kind == "linear":
        return (_plain_matmul(q, s["w"]) * sx.unsqueeze(1) * s["scales"]).to(s["dtype"])
    if kind == "swiglu" and s["gather"]:
        rows = s["perm"].long() // s["top_k"]
        q, sx = q[rows], sx[rows]
    out = []
    for e, (lo, hi) in enumerate(zip(s["bounds"], s["bounds"][1:])):
        if lo == hi:
            continue
        y = _plain_matmul(q[lo:hi], s["w"][e]) * sx[lo:hi].unsqueeze(1) * s["scales"][e]
        if kind == "swiglu":
            g, u = y.chunk(2, dim=1)
            y = _plain_silu(g) * u
        out.append(y)
    return torch.cat(out).to(s["dtype"])


# ---- the framework's calls ------------------------------------------------------------------------------
def _framework():
    path = os.path.join(os.getcwd(), "mini-qwen-llm_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    from mini_qwen_b200 import kernels
    return kernels


def _own(s):
    k = _framework()
    kind, x = s["kind"], s["x"]
    if kind == "quantize":
        q, scale = k.quantize_rows_int8(x)
        return {"q": q, "scale": scale}
    if kind == "linear":
        return k.w8a8_gemm(x, s["w"], s["scales"])
    if kind == "swiglu":
        if s["gather"]:
            return k.w8a8_grouped_swiglu_gather(x, s["perm"], s["top_k"], s["w"], s["scales"], s["offsets"])
        return k.w8a8_grouped_swiglu(x, s["w"], s["scales"], s["offsets"])
    if kind == "down":
        return k.w8a8_grouped_gemm(x, s["w"], s["scales"], s["offsets"])
    if s["experts"] == "dense":
        return k.moe_layer_small(x, s["router"], s["gate_up"], s["down"], s["top_k"], residual=s["residual"])
    if s["experts"] == "w4":
        return k.w4a16_moe_layer_small(x, s["router"], s["gate"], s["up"], s["down"], s["top_k"], GROUP, residual=s["residual"])
    return k.w8a8_moe_layer_small(x, s["router"], (s["gate_up"], s["gate_up_scales"]), (s["down"], s["down_scales"]), s["top_k"],
                                  residual=s["residual"])


@torch.no_grad()
def run(state):
    return _own(state) if own else _plain(state)


# ---- in 64 bits, from the definition --------------------------------------------------------------------
def _exact_rows(x):
    """The quantised rows as numbers, and their scales (stored in 32 bits)."""
    v = x.to(torch.float64)
    scale = torch.div(v.abs().max(dim=1).values, torch.full((), 127.0, dtype=torch.float64, device=v.device))
    scale = scale.to(torch.float32).to(torch.float64)
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(v / safe[:, None]) * (scale != 0)[:, None], scale


def _exact_weight(q, scales):
    return q.to(torch.float64) * scales.to(torch.float64)[..., None]


def _exact_int4(trio, e):
    qw, sc, qz = (t[e] for t in trio)
    q = torch.stack([(qw >> (4 * i)) & 15 for i in range(8)], dim=1).reshape(-1, qw.shape[1]).to(torch.float64)
    z = torch.stack([(qz >> (4 * i)) & 15 for i in range(8)], dim=2).reshape(qz.shape[0], -1).to(torch.float64)
    group = torch.arange(q.shape[0], device=q.device) // GROUP
    return ((q - z[group]) * sc.to(torch.float64)[group]).T


def _swiglu64(a):
    g, u = a[..., :a.shape[-1] // 2], a[..., a.shape[-1] // 2:]
    return g * torch.sigmoid(g) * u


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    kind, x = s["kind"], s["x"]
    if kind == "quantize":
        q, scale = _exact_rows(x)
        return {"q": q.to(torch.int8), "scale": scale}
    if kind == "linear":
        q, scale = _exact_rows(x)
        return (q * scale[:, None]) @ _exact_weight(s["w"], s["scales"]).T
    if kind in ("swiglu", "down"):
        q, scale = _exact_rows(x)
        rows = q * scale[:, None]
        if kind == "swiglu" and s["gather"]:
            rows = rows[torch.div(s["perm"].long(), s["top_k"], rounding_mode="floor")]
        off = s["offsets"].tolist()
        n = s["w"].shape[1] // (2 if kind == "swiglu" else 1)
        out = torch.zeros(rows.shape[0], n, dtype=torch.float64, device=x.device)
        for e in range(len(off) - 1):
            a = rows[off[e]:off[e + 1]] @ _exact_weight(s["w"][e], s["scales"][e]).T
            out[off[e]:off[e + 1]] = _swiglu64(a) if kind == "swiglu" else a
        return out
    p = torch.softmax(x.to(torch.float64) @ s["router"].to(torch.float64).T, dim=1)
    chosen = torch.argsort(p, dim=1, descending=True, stable=True)[:, :s["top_k"]]
    gates = torch.gather(p, 1, chosen)
    gates = gates / gates.sum(dim=1, keepdim=True)
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device) if s["residual"] is None else s["residual"].to(torch.float64)
    if s["experts"] == "w8":
        q, scale = _exact_rows(x)
        rows = q * scale[:, None]
    else:
        rows = x.to(torch.float64)
    for e in sorted(set(chosen.flatten().tolist())):
        tok, slot = torch.nonzero(chosen == e, as_tuple=True)
        if s["experts"] == "dense":
            w1, w2 = s["gate_up"][e].to(torch.float64), s["down"][e].to(torch.float64)
        elif s["experts"] == "w8":
            w1, w2 = _exact_weight(s["gate_up"][e], s["gate_up_scales"][e]), _exact_weight(s["down"][e], s["down_scales"][e])
        else:
            w1, w2 = torch.cat([_exact_int4(s["gate"], e), _exact_int4(s["up"], e)]), _exact_int4(s["down"], e)
        h = _swiglu64(rows[tok] @ w1.T)
        if s["experts"] == "w8":
            step = h.abs().max(dim=1, keepdim=True).values / 127.0
            h = torch.round(h / torch.where(step == 0, torch.ones_like(step), step)) * step
        out = out.index_add(0, tok, (h @ w2.T) * gates[tok, slot][:, None])
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------
def _experts_hit(c):
    """Experts that at least one of the tokens chose, in the mean over experts whose popularity is (rank ** -skew) in odds."""
    E, K, T = c["E"], c["K"], c["T"]
    p = [(r + 1) ** -c.get("skew", 0.0) for r in range(E)]
    total = sum(p)
    return sum(1.0 - (1.0 - min(1.0, K * v / total)) ** T for v in p)


def work(case):
    c = case
    size = DTYPES[c["dtype"]].itemsize
    if c["kind"] == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (size + 1) + 4 * c["rows"], "flops": 4 * n}
    if c["kind"] == "linear":
        M, Kd, N = c["M"], c["Kd"], c["N"]
        return {"bytes": size * M * (Kd + N) + N * Kd + 4 * N, "flops": 2 * M * N * Kd}
    H, E, K, I, T = c["H"], c["E"], c["K"], c["I"], c["T"]
    hit, S = _experts_hit(c), T * K
    if c["kind"] == "swiglu":
        rows = T if c["gather"] else S
        return {"bytes": size * (rows * H + S * I) + hit * (2 * I * H + 8 * I) + 4 * (S + E), "flops": 4 * S * I * H}
    if c["kind"] == "down":
        return {"bytes": size * S * (I + H) + hit * (H * I + 4 * H) + 4 * E, "flops": 2 * S * I * H}
    expert = {"dense": 3 * H * I * size, "w8": 3 * H * I + 8 * I + 4 * H,
              "w4": 3 * (H * I // 2 + (H * I // GROUP) * 5 // 2)}[c["experts"]]
    return {"bytes": hit * expert + E * H * size + size * T * H * (3 if c["residual"] else 2),
            "flops": 6 * S * H * I + 2 * T * H * E}
