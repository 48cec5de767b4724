"""The 4-bit operators and the router, as measured workloads.

Four kinds of case, each one pass of a serving step's operator:

  quant    activations to microscaled 4-bit floating point (NVFP4, MXFP4) and back to their values
  linear   a W4A4 linear layer: quantise the tokens, multiply with a 4-bit weight
  experts  a W4A4 expert product: gather and quantise the routed rows, multiply each with its expert
           (w13 with the gated activation, or w2)
  route    router logits to expert ids and weights, and the expert order of the routed pairs

`run` computes them in plain torch, or, with `own` set, with shard_b200.fp4 and shard_b200.route.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
GROUP = {"nvfp4": 16, "mxfp4": 32}


def listed():
    return [
        # one decode step's hidden state (H of the 4096-wide layers)
        dict(name="quant_nvfp4_token", op="quant", fmt="nvfp4", dtype="bf16", m=1, k=4096, static=False),
        # an odd chunk of activations with a power-of-two scale, from a 16-bit float pipeline
        dict(name="quant_mxfp4_odd_chunk", op="quant", fmt="mxfp4", dtype="fp16", m=1021, k=7168, static=False),
        # a whole prompt batch, one scale per token above the block scales
        dict(name="quant_nvfp4_prompt", op="quant", fmt="nvfp4", dtype="bf16", m=8192, k=7168, static=False),
        # output projection of one decoded token
        dict(name="linear_nvfp4_token", op="linear", fmt="nvfp4", dtype="bf16", out="bf16", m=1, n=4096, k=8192),
        # query projection of a ragged verify chunk, kept in 32 bits
        dict(name="linear_mxfp4_verify", op="linear", fmt="mxfp4", dtype="bf16", out="fp32", m=33, n=32768, k=1024),
        # output projection of a prompt batch
        dict(name="linear_nvfp4_prompt", op="linear", fmt="nvfp4", dtype="bf16", out="bf16", m=8192, n=4096, k=8192),
        # w13 and the gated activation for 16 tokens, top 8 of 64 experts
        dict(name="experts_w13_verify", op="experts", fmt="nvfp4", dtype="bf16", kind="w13", t=16, topk=8, e=64,
             n=4096, k=4096, skew=0.5),
        # w2 of a small layer with a ragged chunk (H 512, I 256)
        dict(name="experts_w2_small", op="experts", fmt="mxfp4", dtype="bf16", kind="w2", t=57, topk=4, e=16, n=512,
             k=256, skew=1.0),
        # w13 of a prompt chunk over a shard of 32 experts
        dict(name="experts_w13_prompt", op="experts", fmt="nvfp4", dtype="bf16", kind="w13", t=2048, topk=8, e=32,
             n=4096, k=4096, skew=0.5),
        # routing of one token: 8 groups, 4 kept, biased sigmoid scores
        dict(name="route_token", op="route", dtype="fp32", t=1, e=256, topk=8, score="sigmoid", bias=True, groups=8,
             kept=4, group_score="top2", masked=0.0, order=False),
        # a ragged chunk of 16-bit logits over 384 experts, softmax without groups
        dict(name="route_softmax_odd", op="route", dtype="bf16", t=1021, e=384, topk=8, score="softmax", bias=False,
             groups=1, kept=1, group_score="max", masked=0.02, order=True),
        # a prompt batch with groups and the expert order that the products read
        dict(name="route_prompt", op="route", dtype="fp32", t=16384, e=256, topk=8, score="sigmoid", bias=True,
             groups=8, kept=4, group_score="top2", masked=0.0, order=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "linear", "experts", "route"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quant":
        k = 32 * _log(rng, 1, 256)
        return dict(op=op, fmt=fmt, dtype=dtype, m=_log(rng, 1, min(16384, 29_000_000 // k)), k=k,
                    static=rng.random() < 0.3)
    if op == "linear":
        m, n, k = _log(rng, 1, 8192), _log(rng, 16, 8192), 32 * _log(rng, 2, 256)
        m = max(1, min(m, (1 << 37) // (n * k)))
        return dict(op=op, fmt=fmt, dtype=dtype, out=rng.choice(["bf16", "fp16", "fp32"]), m=m, n=n, k=k)
    if op == "experts":
        e, n, k = _log(rng, 2, 64), 64 * _log(rng, 2, 64), 32 * _log(rng, 4, 128)
        topk = rng.randint(1, min(8, e))
        t = max(1, min(_log(rng, 1, 2048), (1 << 37) // (topk * n * k)))
        return dict(op=op, fmt=fmt, dtype="bf16", kind=rng.choice(["w13", "w2"]), t=t, topk=topk, e=e, n=n, k=k,
                    skew=round(rng.uniform(0.0, 1.0), 2))
    groups = rng.choice([1, 1, 2, 4, 8, 16])
    e = groups * _log(rng, max(2, 16 // groups), 512 // groups)
    kept = rng.randint(max(1, groups // 2), groups)
    topk = min(rng.randint(1, 12), kept * (e // groups))
    return dict(op=op, dtype=dtype, t=_log(rng, 1, 8192), e=e, topk=topk,
                score=rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]), bias=rng.random() < 0.6, groups=groups,
                kept=kept, group_score=rng.choice(["max", "top2"]), masked=rng.choice([0.0, 0.05]),
                order=rng.random() < 0.7)


# ── inputs ─────────────────────────────────────────────────────────────────────────────────────

def _activations(g, rows, k, dtype):
    """Tokens after a norm: unit values with a spread of channel sizes and a few large channels."""
    ch = torch.exp(0.4 * torch.randn(k, generator=g, device=DEV))
    ch = torch.where(torch.rand(k, generator=g, device=DEV) < 0.004, 12 * ch, ch)
    return (torch.randn(rows, k, generator=g, device=DEV) * ch).to(DTYPES[dtype])


def _weights(g, fmt, mats, n, k):
    """Canonical 4-bit weights [mats, N, K]: packed e2m1 codes (low nibble first), block scales as bytes,
    fp32 tensor scales [mats, 2] (w1 and w3, or the same twice). Codes and scales have the distribution
    that quantising normal weights gives."""
    pairs = torch.randn(1 << 14, 2, generator=g, device=DEV) * 2.6
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    code = torch.bucketize(pairs.abs(), mids) + 8 * (pairs < 0)
    table = (code[:, 0] + 16 * code[:, 1]).to(torch.uint8)
    codes = table[torch.randint(0, 1 << 14, (mats, n, k // 2), generator=g, device=DEV, dtype=torch.int32)]
    shape = (mats, n, k // GROUP[fmt])
    if fmt == "nvfp4":
        s = (448 * (0.36 + 0.07 * torch.randn(shape, generator=g, device=DEV)).clamp(0.05, 1.0))
        scales = s.to(torch.float8_e4m3fn).view(torch.uint8)
        ts = 4e-5 * (1 + torch.rand(mats, 2, generator=g, device=DEV))
    else:
        scales = torch.randint(119, 122, shape, generator=g, device=DEV, dtype=torch.uint8)
        ts = None
    return codes, scales, ts


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "route":
        logits = 1.5 * torch.randn(case["t"], case["e"], generator=g, device=DEV)
        if case["masked"]:
            logits.masked_fill_(torch.rand(logits.shape, generator=g, device=DEV) < case["masked"], -math.inf)
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        s["bias_t"] = 0.1 * torch.randn(case["e"], generator=g, device=DEV) if case["bias"] else None
        return s
    fmt, k = case["fmt"], case["k"]
    if case["op"] == "quant":
        s["x"] = _activations(g, case["m"], k, case["dtype"])
        s["ts"] = torch.full((1,), 40.0 / 2688, device=DEV) if case["static"] and fmt == "nvfp4" else None
        return s
    mats = case.get("e", 1)
    s["codes"], s["scales"], ts = _weights(g, fmt, mats, case["n"], k)
    s["ts"] = ts if case.get("kind") == "w13" or ts is None else ts[:, :1].contiguous()
    if case["op"] == "linear":
        s["x"] = _activations(g, case["m"], k, case["dtype"])
    else:
        t, topk = case["t"], case["topk"]
        s["x"] = _activations(g, t if case["kind"] == "w13" else t * topk, k, case["dtype"])
        pop = torch.exp(case["skew"] * torch.randn(mats, generator=g, device=DEV))
        ids = torch.multinomial(pop.expand(t, mats), topk, generator=g).reshape(-1)
        order = torch.sort(ids, stable=True).indices
        s["rows"] = (order // topk if case["kind"] == "w13" else order).to(torch.int32)
        count = torch.bincount(ids, minlength=mats)
        s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
        s["most"] = int(count.max())
    if own:  # a user's program lays its weights out once, at load time
        from shard_b200 import fp4
        kind = fp4.W13 if case.get("kind") == "w13" else fp4.PLAIN
        one = (lambda v: v) if case["op"] == "experts" else (lambda v: None if v is None else v[0])
        s["operand"] = fp4.pack(fmt, one(s["codes"]), one(s["scales"]), one(s["ts"]), kind=kind)
    return s


# ── the plain form ─────────────────────────────────────────────────────────────────────────────

def _e2m1_round(v):
    """Nearest e2m1 value of |v| <= 6, ties to the even code."""
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return torch.round(v / step) * step


def _e4m3_round(v):
    """Nearest e4m3 value of 0 <= v <= 448, ties to even."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp_min(-9))
    return torch.round(v / step) * step


def _quantised(x, fmt, ts):
    """The values that quantised rows stand for, in 64 bits (borders are compared there)."""
    m, k = x.shape
    v = x.double().reshape(m, -1, GROUP[fmt])
    amax = v.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        mant, e = torch.frexp(amax.clamp_min(6 * 2.0 ** -126))
        s = torch.ldexp(torch.ones_like(amax), torch.where(mant <= 0.75, e - 3, e - 2))
    else:
        t = (amax.amax(1, keepdim=True) / 2688).clamp_min(2.0 ** -126).float().double() if ts is None else ts.double()
        s = _e4m3_round((amax / (6 * t)).clamp_max(448.0)) * t
    q = _e2m1_round((v / torch.where(s > 0, s, 1.0)).clamp(-6, 6))
    return (q * s).reshape(m, k)


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _weight_values(s):
    """fp32 [mats, N, K] of the canonical weights."""
    table = torch.tensor(_E2M1, device=DEV)
    c = s["codes"].int()
    mats, n, k2 = c.shape
    v = torch.stack([table[c & 15], table[c >> 4]], -1).reshape(mats, n, -1, GROUP[s["fmt"]])
    if s["fmt"] == "nvfp4":
        sc = s["scales"].view(torch.float8_e4m3fn).float()
        halves = s["ts"].shape[1]
        sc = (sc.reshape(mats, halves, n // halves, -1) * s["ts"][:, :, None, None]).reshape(sc.shape)
    else:
        sc = torch.ldexp(torch.ones(s["scales"].shape, device=DEV), s["scales"].int() - 127)
    return (v * sc[..., None]).reshape(mats, n, 2 * k2)


def _plain_route(s):
    l = s["logits"].double()
    masked = torch.isinf(l) & (l < 0)
    if s["score"] == "softmax":
        score = torch.exp(l - l.amax(1, keepdim=True).clamp_min(-1e300))
        score = score / score.sum(1, keepdim=True).clamp_min(1e-300)
    elif s["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-l))
    else:
        score = torch.sqrt(torch.where(l > 0, l, 0.0) + torch.log1p(torch.exp(-l.abs())))
    score = torch.where(masked, 0.0, score)
    t, e = l.shape
    pick = torch.where(masked, -math.inf, l if s["bias_t"] is None else score + s["bias_t"].double())
    if s["groups"] > 1:
        size = e // s["groups"]
        if s["group_score"] == "top2":
            two = pick if s["bias_t"] is not None else torch.where(masked, -math.inf, score)
            best = torch.sort(two.reshape(t, -1, size), -1, descending=True).values[..., :2]
            gs = torch.where(best == -math.inf, 0.0, best).sum(-1)
            gs = torch.where(best[..., 0] == -math.inf, -math.inf, gs)
        else:
            gs = pick.reshape(t, -1, size).amax(-1)
        rank = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, : s["kept"]]
        keep = torch.zeros_like(gs, dtype=torch.bool).scatter(1, rank, True).repeat_interleave(size, 1)
        first = torch.where(keep, 0, 1)  # a masked expert of a kept group comes before any of the others
        pick = torch.where(keep, pick, -math.inf)
    else:
        first = torch.zeros_like(pick, dtype=torch.long)
    by_pick = torch.sort(pick, dim=1, descending=True, stable=True).indices
    by_both = torch.sort(first.gather(1, by_pick), dim=1, stable=True).indices
    ids = by_pick.gather(1, by_both)[:, : s["topk"]].contiguous()
    w = score.gather(1, ids)
    w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return w.float(), ids


def _plain_order(ids, e):
    """(offsets [E+1], tokens in expert order, place of each pair in that order)."""
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(order).scatter(0, order, torch.arange(order.numel(), device=DEV))
    count = torch.zeros(e, dtype=torch.long, device=DEV).scatter_add(0, flat, torch.ones_like(flat))
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    return offsets.int(), (order // ids.shape[1]).int(), place.reshape(ids.shape).int()


def _plain(s):
    if s["op"] == "route":
        w, ids = _plain_route(s)
        return (w, ids) + (_plain_order(ids, s["e"]) if s["order"] else ())
    if s["op"] == "quant":
        return _quantised(s["x"], s["fmt"], s["ts"]).to(s["x"].dtype)
    w = _weight_values(s)
    if s["op"] == "linear":
        return (_quantised(s["x"], s["fmt"], None).float() @ w[0].T).to(DTYPES[s["out"]])
    a = _quantised(s["x"][s["rows"].long()], s["fmt"], None).float()
    a = torch.cat([a, a.new_zeros(1, a.shape[1])])
    at = s["offsets"][:-1, None].long() + torch.arange(s["most"], device=DEV)
    at = torch.where(at < s["offsets"][1:, None], at, a.shape[0] - 1)
    o = torch.bmm(a[at], w.transpose(1, 2))
    if s["kind"] == "w13":
        gate, up = o.chunk(2, -1)
        o = gate / (1 + torch.exp(-gate)) * up
    y = o.new_empty(a.shape[0], o.shape[-1])
    y[at.reshape(-1)] = o.reshape(-1, o.shape[-1])
    return y[:-1].to(torch.bfloat16)


def run(s):
    if not own:
        return _plain(s)
    from shard_b200 import fp4, route
    if s["op"] == "quant":
        return fp4.dequant(fp4.quant(s["x"], s["fmt"], tensor_scale=s["ts"]), s["x"].dtype)
    if s["op"] == "linear":
        return fp4.gemm(fp4.quant(s["x"], s["fmt"]), s["operand"], out_dtype=DTYPES[s["out"]])
    if s["op"] == "experts":
        a = fp4.quant(s["x"], s["fmt"], rows=s["rows"], offsets=s["offsets"])
        return fp4.grouped_gemm(a, s["operand"])
    w, ids = route.topk(s["logits"], s["topk"], bias=s["bias_t"], score=s["score"], n_group=s["groups"],
                        topk_group=s["kept"], group_score=s["group_score"])
    if not s["order"]:
        return w, ids
    o = route.expert_order(ids, s["e"])
    return w, ids, o.offsets, o.tokens, o.places


def work(case):
    op = case["op"]
    if op == "route":
        t, e, k = case["t"], case["e"], case["topk"]
        b = t * e * SIZE[case["dtype"]] + 12 * t * k + (4 * e if case["bias"] else 0)
        return {"bytes": b + (8 * t * k + 4 * (e + 1) if case["order"] else 0), "flops": 8 * t * e}
    k, c = case["k"], 0.5 + 1.0 / GROUP[case["fmt"]]
    if op == "quant":
        return {"bytes": 2 * case["m"] * k * SIZE[case["dtype"]], "flops": 8 * case["m"] * k}
    if op == "linear":
        m, n = case["m"], case["n"]
        return {"bytes": m * k * SIZE[case["dtype"]] + n * k * c + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    t, p, e, n = case["t"], case["t"] * case["topk"], case["e"], case["n"]
    hit = e * (1 - (1 - 1 / e) ** p)  # experts that at least one pair reaches
    x = (t if case["kind"] == "w13" else p) * k * SIZE[case["dtype"]]
    return {"bytes": x + hit * n * k * c + 2 * p * (n // 2 if case["kind"] == "w13" else n) + 4 * p,
            "flops": 2 * p * n * k}


# ── the definition in 64 bits, in other steps ──────────────────────────────────────────────────

_VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
_E4M3 = np.array([(m / 8) * 2.0 ** -6 for m in range(8)]
                 + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])


def _nearest(v, values):
    """The nearest of `values` (ascending; neighbours' borders to the even index), for v >= 0."""
    vals = torch.tensor(values, device=v.device, dtype=torch.float64)
    mid = (vals[1:] + vals[:-1]) / 2
    lo, hi = torch.bucketize(v, mid), torch.bucketize(v, mid, right=True)
    return vals[torch.where(lo % 2 == 0, lo, hi)]


def _exact_values(x, fmt, ts):
    v = x.to(torch.float64)
    blocks = v.view(v.shape[0], v.shape[1] // GROUP[fmt], GROUP[fmt])
    top = blocks.abs().max(2).values
    if fmt == "mxfp4":
        s = torch.exp2(torch.ceil(torch.log2(top.clamp_min(6 * 2.0 ** -126) / 6) - 1e-13))
    else:
        t = ts.double() if ts is not None else (top.max(1).values / 2688).float().double().clamp_min(2.0 ** -126)[:, None]
        s = _nearest((top / t / 6).clamp_max(448), _E4M3) * t
    s = s[:, :, None]
    mag = torch.where(s > 0, blocks.abs() / s, torch.zeros_like(blocks)).clamp_max(6)
    return (_nearest(mag, _VALUES) * s * torch.sign(blocks)).view(v.shape)


def _exact_weight(s, mat):
    codes = s["codes"][mat].long()
    sign = lambda c: 1.0 - 2.0 * (c >= 8).double()  # noqa: E731
    vals = torch.tensor(_VALUES, device=DEV)
    low, high = codes % 16, codes // 16
    w = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=DEV)
    w[:, 0::2], w[:, 1::2] = vals[low % 8] * sign(low), vals[high % 8] * sign(high)
    if s["fmt"] == "nvfp4":
        sc = torch.tensor(np.append(_E4M3, np.nan), device=DEV)[s["scales"][mat].long()]
        rows = sc.shape[0] // s["ts"].shape[1]
        for h in range(s["ts"].shape[1]):
            sc[h * rows:(h + 1) * rows] *= s["ts"][mat, h].double()
    else:
        sc = torch.pow(2.0, s["scales"][mat].double() - 127)
    return w * sc.repeat_interleave(GROUP[s["fmt"]], 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        return _exact_values(s["x"], s["fmt"], s["ts"])
    if case["op"] == "linear":
        return _exact_values(s["x"], s["fmt"], None) @ _exact_weight(s, 0).T
    if case["op"] == "experts":
        x, rows, off, parts = s["x"], s["rows"].long(), s["offsets"].tolist(), []
        for e in range(case["e"]):
            if off[e + 1] > off[e]:
                o = _exact_values(x[rows[off[e]:off[e + 1]]], s["fmt"], None) @ _exact_weight(s, e).T
                half = o.shape[1] // 2
                parts.append(o[:, :half] * torch.sigmoid(o[:, :half]) * o[:, half:] if s["kind"] == "w13" else o)
        return torch.cat(parts)
    # weights: each chosen expert's score over the sum of the chosen ones; ids are whole numbers
    l = s["logits"].double().cpu().numpy()
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if case["score"] == "softmax":
            p = np.exp(l - l.max(1, keepdims=True))
            p = np.nan_to_num(p / p.sum(1, keepdims=True))
        elif case["score"] == "sigmoid":
            p = np.exp(-np.logaddexp(0, -l))
        else:
            p = np.sqrt(np.logaddexp(0, l))
    off = np.isneginf(l)
    pick = l if s["bias_t"] is None else p + s["bias_t"].double().cpu().numpy()
    w = np.empty((case["t"], case["topk"]))
    size = case["e"] // case["groups"]
    for i in range(case["t"]):
        v = np.where(off[i], -np.inf, pick[i])
        allowed = np.arange(case["e"])
        if case["groups"] > 1:
            gv = v if s["bias_t"] is not None or case["group_score"] == "max" else np.where(off[i], -np.inf, p[i])
            top = -np.sort(-gv.reshape(-1, size), 1)[:, : 2 if case["group_score"] == "top2" else 1]
            gs = np.where(np.isneginf(top[:, 0]), -np.inf, np.where(np.isneginf(top), 0, top).sum(1))
            kept = np.sort(np.argsort(-gs, kind="stable")[: case["kept"]])
            allowed = (kept[:, None] * size + np.arange(size)).reshape(-1)
        ids = allowed[np.argsort(-v[allowed], kind="stable")[: case["topk"]]]
        c = np.where(off[i][ids], 0, p[i][ids])
        w[i] = c / c.sum() if c.sum() > 0 else 0
    w = torch.from_numpy(w)
    return (w, None) + ((None, None, None) if case["order"] else ())
