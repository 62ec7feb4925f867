"""What is timed of the block-scaled FP8 operators and the expert routing.

Four operators, each in its plain form (elementary torch operations) and, with ``own`` true, as the framework's
entry points compute it:

* ``route``    expert choice from router logits: softmax or sigmoid scores, a selection bias, expert groups, top-k
               with ties to the lowest index, renormalised weights. ``gpu.routing.route_topk``.
* ``quant``    FP8 (e4m3) values with one f32 scale per 128 of a row (activations) or per 128 x 128 block (weights).
               ``gpu.quant.quantize_fp8_activation_blocks`` / ``quantize_3d_to_fp8_block``.
* ``linear``   y = x W^T with W in 128 x 128-block FP8 and x quantized per 128 of a row in the call.
               ``gpu.fp8_block_matmul.fp8_block_linear``.
* ``experts``  the routed experts' gated MLP with such weights, gate_up, activation, re-quantization, down and the
               weighted sum over a token's experts. ``bridges.gemma4.moe_ops.fp8_block_experts``.

The quantizer of all four: with a = max(max|x| over the block, 1e-30), scale = f32(a / 448), inv = f32(448 / a),
q = e4m3(f32(x * inv)), the value is q * scale. A block that holds an infinity or a NaN has a NaN scale.
"""
import functools
import math

import numpy as np
import torch

own = False

BLOCK = 128
F8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@functools.lru_cache(None)
def _entry():
    """The framework's entry points (only where ``own`` is true)."""
    import os
    import sys
    package = os.path.join(os.getcwd(), "aeo-quant_b200")
    if package not in sys.path:
        sys.path.insert(1, package)
    from aeo_quant_b200.bridges.gemma4 import moe_ops
    from aeo_quant_b200.gpu import fp8_block_matmul, quant, routing
    return {"route": routing.route_topk, "rows": quant.quantize_fp8_activation_blocks,
            "blocks": quant.quantize_3d_to_fp8_block, "linear": fp8_block_matmul.fp8_block_linear,
            "experts": moe_ops.fp8_block_experts}


# ------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of the 128-expert decoder: latency alone
        dict(op="route", name="route_one_token", T=1, E=128, k=8, score="softmax", dtype="bf16", bias=False,
             groups=1, kept=1, group_score="max", renorm=True, scale=1.0, masked=0.0),
        # a prefill chunk, sigmoid scores with a balance bias and grouped choice
        dict(op="route", name="route_grouped_4k", T=4096, E=256, k=8, score="sigmoid", dtype="f32", bias=True,
             groups=8, kept=4, group_score="top2", renorm=True, scale=2.5, masked=0.01),
        # the largest batch the expert-parallel layer takes: 32 sequences of 2048 tokens
        dict(op="route", name="route_softmax_64k", T=65536, E=128, k=8, score="softmax", dtype="bf16", bias=False,
             groups=1, kept=1, group_score="max", renorm=True, scale=1.0, masked=0.0),
        # activations of a prefill in front of a linear layer
        dict(op="quant", name="quant_rows_32k", kind="rows", E=1, M=32768, K=2816, dtype="bf16"),
        # a few rows with a ragged last block: one step of a small batch
        dict(op="quant", name="quant_rows_small", kind="rows", E=1, M=17, K=704, dtype="f32"),
        # a stack of expert weights while a checkpoint is converted (the gate_up of 32 experts)
        dict(op="quant", name="quant_weights_32x", kind="blocks", E=32, M=1408, K=2816, dtype="bf16"),
        # one token through one projection: latency and the weight's bytes
        dict(op="linear", name="linear_one_token", M=1, N=1408, K=2816, out="bf16"),
        # a decode batch through a dense MLP whose width is not a multiple of 128
        dict(op="linear", name="linear_batch_48", M=48, N=2112, K=2816, out="bf16"),
        # a prefill of 16 sequences of 2048 tokens
        dict(op="linear", name="linear_32k", M=32768, N=1408, K=2816, out="bf16"),
        # one decoded token: eight experts' weights are the work
        dict(op="experts", name="experts_one_token", T=1, E=128, k=8, H=2816, I=704, act="gelu_pytorch_tanh",
             dropped=0.0),
        # a padded decode batch: some slots carry no expert
        dict(op="experts", name="experts_batch_16", T=16, E=128, k=8, H=2816, I=704, act="silu", dropped=0.1),
        # prefill of 4096 tokens over 128 experts
        dict(op="experts", name="experts_4k", T=4096, E=128, k=8, H=2816, I=704, act="gelu_pytorch_tanh",
             dropped=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "quant", "linear", "linear", "experts", "experts"])
    if op == "route":
        E = rng.choice([rng.randint(2, 24), 16 * rng.randint(2, 32), 128, 256])
        groups = rng.choice([1, 1] + [g for g in (2, 4, 8, 16) if E % g == 0 and E // g >= 2])
        kept = rng.randint(1, groups)
        k = rng.randint(1, min(16, E // groups * kept))
        return dict(op=op, T=_log(rng, 1, 32768), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.5, groups=groups, kept=kept,
                    group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), masked=rng.choice([0.0, 0.05]))
    if op == "quant":
        kind = rng.choice(["rows", "blocks"])
        K = rng.choice([16 * rng.randint(1, 512), rng.randint(1, 4096)])
        if kind == "rows":
            return dict(op=op, kind=kind, E=1, M=_log(rng, 1, min(32768, 92_000_000 // K)), K=K,
                        dtype=rng.choice(["bf16", "f16", "f32"]))
        E = _log(rng, 1, 32)
        return dict(op=op, kind=kind, E=E, M=_log(rng, 1, min(4096, 60_000_000 // (K * E))), K=K,
                    dtype=rng.choice(["bf16", "f32"]))
    if op == "linear":
        N, K = _log(rng, 16, 8192), 16 * _log(rng, 4, 512)
        return dict(op=op, M=_log(rng, 1, min(32768, 120_000_000_000 // (N * K))), N=N, K=K,
                    out=rng.choice(["bf16", "bf16", "f32"]))
    E, H, I = _log(rng, 2, 128), 16 * _log(rng, 16, 176), 64 * rng.randint(1, 16)
    k = rng.randint(1, min(8, E))
    return dict(op=op, T=_log(rng, 1, 4096), E=E, k=k, H=H, I=I, act=rng.choice(["gelu_pytorch_tanh", "silu"]),
                dropped=rng.choice([0.0, 0.1]))


# ------------------------------------------------------------------------------------------------- the inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, width):
    """Hidden states: unit normal, one channel in 64 fifteen times as large (outlier channels)."""
    gain = torch.where(torch.rand(width, generator=g, device="cuda") < 1 / 64, 15.0, 1.0)
    return _randn(g, rows, width) * gain


def _weights(g, E, N, K):
    """Weights of std 0.02 in the checkpoint's form: e4m3 values and one f32 scale per 128 x 128 block."""
    q = torch.empty(E, N, K, dtype=F8, device="cuda")
    s = torch.empty(E, -(-N // BLOCK), -(-K // BLOCK), device="cuda")
    for e in range(0, E, 16):
        w = (_randn(g, min(16, E - e), N, K) * 0.02).to(torch.bfloat16)
        q[e:e + 16], s[e:e + 16] = _quantize_blocks(w)
    return q, s


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        logits = _randn(g, T, E) * 1.5
        if case["masked"]:
            logits.masked_fill_(torch.rand(T, E, generator=g, device="cuda") < case["masked"], -math.inf)
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        s["bias"] = _randn(g, E) * 0.05 if case["bias"] else None
    elif case["op"] == "quant":
        if case["kind"] == "rows":
            s["x"] = _activations(g, case["M"], case["K"]).to(DTYPES[case["dtype"]])
        else:
            s["x"] = (_randn(g, case["E"], case["M"], case["K"]) * 0.02).to(DTYPES[case["dtype"]])
    elif case["op"] == "linear":
        s["x"] = _activations(g, case["M"], case["K"]).to(torch.bfloat16)
        q, sc = _weights(g, 1, case["N"], case["K"])
        s["w"], s["w_scale"] = q[0], sc[0]
    else:
        T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
        s["x"] = _activations(g, T, H).to(torch.bfloat16)
        # a popular expert draws up to e times as many tokens as an average one
        taste = torch.rand(E, generator=g, device="cuda")
        scores = torch.rand(T, E, generator=g, device="cuda").log().neg().log().neg() + taste
        ids = scores.topk(k, dim=-1).indices
        w = torch.softmax(_randn(g, T, k), -1)
        if case["dropped"]:
            ids = ids.masked_fill(torch.rand(T, k, generator=g, device="cuda") < case["dropped"], E)
        s["ids"], s["weights"] = ids, w
        s["gate_up"], s["gate_up_scale"] = _weights(g, E, 2 * I, H)
        s["down"], s["down_scale"] = _weights(g, E, H, I)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _pad(x, *dims):
    """x with zeros up to multiples of 128 along the given (negative) dimensions."""
    pads = [0, 0] * max(-d for d in dims)
    for d in dims:
        pads[2 * (-d - 1) + 1] = -x.shape[d] % BLOCK
    return torch.nn.functional.pad(x, pads)


def _code(x, amax):
    """(e4m3 values of x * inv, scale) for the block maxima `amax` (keepdim of x)."""
    top = torch.full_like(amax, 448.0)
    amax = torch.where(amax.isfinite(), amax.clamp_min(1e-30), math.nan)
    return (x * (top / amax)).to(F8), amax / top


def _quantize_rows(x):
    M, K = x.shape
    v = _pad(x.float(), -1).view(M, -1, BLOCK)
    q, s = _code(v, v.abs().amax(-1, keepdim=True))
    return q.view(M, -1)[:, :K].contiguous(), s.view(M, -1)


def _quantize_blocks(w):
    E, N, K = w.shape
    v = _pad(w.float(), -1, -2)
    v = v.view(E, v.shape[1] // BLOCK, BLOCK, v.shape[2] // BLOCK, BLOCK)
    q, s = _code(v, v.abs().amax((2, 4), keepdim=True))
    return q.view(E, v.shape[1] * BLOCK, -1)[:, :N, :K].contiguous(), s.view(E, v.shape[1], -1)


def _values_rows(q, s):
    return q.float() * s.repeat_interleave(BLOCK, -1)[..., : q.shape[-1]]


def _values_blocks(q, s):
    N, K = q.shape[-2:]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]


def _activation(name, x):
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def _route_plain(s):
    c, l = s["case"], s["logits"].double()       # 64 bits: the order of close scores decides a whole number
    T, E = l.shape
    if c["score"] == "softmax":
        top = l.amax(-1, keepdim=True)
        p = torch.exp(l - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        score = torch.where(total > 0, p / total, 0.0)
    else:
        score = 1 / (1 + torch.exp(-l))
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = choice.masked_fill(l == -math.inf, -math.inf)
    if c["groups"] > 1:
        g = choice.view(T, c["groups"], -1)
        best = g.sort(dim=-1, descending=True).values[..., :2]
        best = best[..., 0] + (best[..., 1].masked_fill(best[..., 1] == -math.inf, 0.0) if c["group_score"] == "top2"
                               else 0.0)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["kept"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = g.masked_fill(~keep[..., None], -math.inf).view(T, E)
    value, ids = choice.sort(dim=-1, descending=True, stable=True)
    value, ids = value[:, : c["k"]], ids[:, : c["k"]]
    empty = value == -math.inf                   # fewer experts left than slots: no expert, weight 0
    w = score.gather(1, ids).masked_fill(empty, 0.0)
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return (w * c["scale"]).float(), ids.masked_fill(empty, E)


def _experts_plain(s):
    c, x, ids = s["case"], s["x"], s["ids"]
    T, E, k = c["T"], c["E"], c["k"]
    P = T * k
    xd = _values_rows(*_quantize_rows(x))
    flat = ids.reshape(-1)
    valid = (flat >= 0) & (flat < E)
    expert = torch.where(valid, flat, 0)
    pair_x = xd.repeat_interleave(k, 0)
    if P <= 128:                                 # the chosen experts' weights, one copy for each pair
        gu = _values_blocks(s["gate_up"].view(torch.uint8)[expert].view(F8), s["gate_up_scale"][expert])
        g, u = torch.bmm(gu, pair_x[:, :, None])[..., 0].chunk(2, -1)
        hd = _values_rows(*_quantize_rows(_activation(c["act"], g) * u))
        del gu
        dw = _values_blocks(s["down"].view(torch.uint8)[expert].view(F8), s["down_scale"][expert])
        y = torch.bmm(dw, hd[:, :, None])[..., 0]
    else:                                        # tokens in padded rows of their experts
        hot = (torch.nn.functional.one_hot(expert, E) * valid[:, None]).to(torch.int32)
        at = (hot.cumsum(0) - hot).gather(1, expert[:, None])[:, 0].long()
        room = int(hot.sum(0).max())
        at = torch.where(valid, at, room)        # pairs without an expert share a row that is not used
        rows = torch.zeros(E, room + 1, x.shape[1], device=x.device)
        rows[expert, at] = pair_x
        g, u = torch.bmm(rows, _values_blocks(s["gate_up"], s["gate_up_scale"]).transpose(1, 2)).chunk(2, -1)
        h = _activation(c["act"], g) * u
        hd = _values_rows(*_quantize_rows(h.reshape(E * (room + 1), -1))).view(E, room + 1, -1)
        y = torch.bmm(hd, _values_blocks(s["down"], s["down_scale"]).transpose(1, 2))[expert, at]
    y = torch.where(valid[:, None], y * s["weights"].reshape(-1, 1), 0.0)
    return y.view(T, k, -1).sum(1).to(torch.bfloat16)


def run(state):
    c, op = state["case"], state["op"]
    if own:
        f = _entry()
        if op == "route":
            return f["route"](state["logits"], c["k"], score=c["score"], bias=state["bias"], n_group=c["groups"],
                              topk_group=c["kept"], group_score=c["group_score"], renormalize=c["renorm"],
                              scale=c["scale"])
        if op == "quant":
            return f[c["kind"]](state["x"])
        if op == "linear":
            return f["linear"](state["x"], state["w"], state["w_scale"], out_dtype=DTYPES[c["out"]])
        return f["experts"](state["x"], state["ids"], state["weights"], state["gate_up"], state["gate_up_scale"],
                            state["down"], state["down_scale"], activation=c["act"])
    if op == "route":
        return _route_plain(state)
    if op == "quant":
        return _quantize_rows(state["x"]) if c["kind"] == "rows" else _quantize_blocks(state["x"])
    if op == "linear":
        y = _values_rows(*_quantize_rows(state["x"])) @ _values_blocks(state["w"], state["w_scale"]).t()
        return y.to(DTYPES[c["out"]])
    return _experts_plain(state)


# ----------------------------------------------------------------------------------------------------- work

def work(case):
    c, size = case, {"bf16": 2, "f16": 2, "f32": 4}
    up = lambda n: -(-n // BLOCK)  # noqa: E731
    if c["op"] == "route":
        return {"bytes": c["T"] * (c["E"] * size[c["dtype"]] + c["k"] * 12) + (4 * c["E"] if c["bias"] else 0),
                "flops": 8 * c["T"] * c["E"]}
    if c["op"] == "quant":
        n = c["E"] * c["M"] * c["K"]
        scales = c["M"] * up(c["K"]) if c["kind"] == "rows" else c["E"] * up(c["M"]) * up(c["K"])
        return {"bytes": n * (size[c["dtype"]] + 1) + 4 * scales, "flops": 3 * n}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": 2 * M * K + N * K + 4 * up(N) * up(K) + size[c["out"]] * M * N, "flops": 2 * M * N * K}
    T, E, k, H, I = (c[n] for n in ("T", "E", "k", "H", "I"))
    pairs = T * k * (1 - c["dropped"])
    used = E * (1 - (1 - 1 / E) ** pairs) if T > 1 else min(E, pairs)   # experts that any token chose
    per = 3 * H * I + 4 * (up(2 * I) * up(H) + up(H) * up(I))
    return {"bytes": used * per + 4 * T * H + 12 * T * k, "flops": 6 * pairs * H * I}


# ----------------------------------------------------------------------------------------------------- exact

def _code64(v, a):
    """The quantizer's values of v (64 bits) for the block maximum a: the scale and its inverse are f32 by
    definition, their product with the input is rounded to f32 once."""
    a = a.clamp_min(float(np.float32(1e-30)))
    inv, scale = (448.0 / a).float().double(), (a / 448.0).float().double()
    p = (v * inv).float().double()
    mag = p.abs()
    e = torch.floor(torch.log2(mag.clamp_min(2.0 ** -9))).clamp(-6, 8)
    e = torch.where(torch.exp2(e + 1) <= mag, e + 1, e)          # log2 may round across a power of two
    e = torch.where((torch.exp2(e) > mag) & (e > -6), e - 1, e)
    step = torch.exp2(e - 3)
    return torch.sign(p) * torch.minimum(torch.round(mag / step) * step, torch.full_like(mag, 448.0)), scale


def _rows64(x):
    """(values of the codes, values, scales) of rows cut into 128s, block by block."""
    q, d, s = torch.empty_like(x), torch.empty_like(x), []
    for b in range(0, x.shape[1], BLOCK):
        v = x[:, b:b + BLOCK]
        c, sc = _code64(v, v.abs().amax(1, keepdim=True))
        q[:, b:b + BLOCK], d[:, b:b + BLOCK] = c, c * sc
        s.append(sc)
    return q, d, torch.cat(s, 1)


def _weight64(q, s):
    w = q.double()
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= s[i, j].double()
    return w


def _act64(name, x):
    if name == "silu":
        return x * torch.sigmoid(x)
    return torch.nn.functional.gelu(x, approximate="tanh")


def _route64(s):
    c = s["case"]
    l = s["logits"].double().cpu().numpy()
    b = np.zeros(l.shape[1]) if s["bias"] is None else s["bias"].double().cpu().numpy()
    T, E = l.shape
    masked = np.isneginf(l)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        if c["score"] == "softmax":
            p = np.exp(l - np.where(masked.all(1), 0.0, l.max(1))[:, None])
            score = np.where(masked.all(1)[:, None], 0.0, p / p.sum(1, keepdims=True))
        else:
            score = 1.0 / (1.0 + np.exp(-l))
    choice = np.where(masked, -np.inf, score + b)
    if c["groups"] > 1:
        per = E // c["groups"]
        worth = np.empty((T, c["groups"]))
        for g in range(c["groups"]):
            v = -np.sort(-choice[:, g * per:(g + 1) * per], 1)
            worth[:, g] = v[:, 0]
            if c["group_score"] == "top2" and per > 1:
                worth[:, g] += np.where(np.isneginf(v[:, 1]), 0.0, v[:, 1])
        order = np.argsort(-worth, 1, kind="stable")
        for r in range(c["kept"], c["groups"]):
            for g in range(c["groups"]):
                choice[order[:, r] == g, g * per:(g + 1) * per] = -np.inf
    ids = np.argsort(-choice, 1, kind="stable")[:, : c["k"]]
    none = np.isneginf(np.take_along_axis(choice, ids, 1))
    w = np.where(none, 0.0, np.take_along_axis(score, ids, 1))
    if c["renorm"]:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return w * c["scale"], np.where(none, E, ids).astype(np.int64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _route64(s)
    if case["op"] == "quant":
        x = s["x"].double()
        if case["kind"] == "rows":
            q, _, sc = _rows64(x)
            return q, sc
        E, N, K = x.shape
        q, sc = torch.empty_like(x), torch.empty(E, -(-N // BLOCK), -(-K // BLOCK), dtype=torch.float64,
                                                 device=x.device)
        for i in range(sc.shape[1]):
            for j in range(sc.shape[2]):
                v = x[:, i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK]
                cq, cs = _code64(v, v.abs().amax((1, 2), keepdim=True))
                q[:, i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] = cq
                sc[:, i, j] = cs[:, 0, 0]
        return q, sc
    if case["op"] == "linear":
        return _rows64(s["x"].double())[1] @ _weight64(s["w"], s["w_scale"]).t()
    T, E = case["T"], case["E"]
    x = _rows64(s["x"].double())[1]
    out = torch.zeros(T, x.shape[1], dtype=torch.float64, device=x.device)
    for e in range(E):
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        g, u = (x[t] @ _weight64(s["gate_up"][e], s["gate_up_scale"][e]).t()).chunk(2, 1)
        h = _rows64(_act64(case["act"], g) * u)[1]
        y = h @ _weight64(s["down"][e], s["down_scale"][e]).t()
        out.index_add_(0, t, y * s["weights"][t, j].double()[:, None])
    return out
