"""Plain 64-bit forms of shard_b200.fp4 and shard_b200.route for their tests, on the CPU."""
import math

import torch

from shard_b200 import formats as F

MAGS = torch.tensor(F.E2M1, dtype=torch.float64)
MIDS = torch.tensor(F.E2M1_MID, dtype=torch.float64)
E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest(v, values):
    """Index of the nearest of ascending `values` to v >= 0, ties to the even index."""
    mid = (values[1:] + values[:-1]) / 2
    lo, hi = torch.bucketize(v, mid), torch.bucketize(v, mid, right=True)
    return torch.where(lo % 2 == 0, lo, hi).clamp_max(len(values) - 1)


def quant(x, fmt, ts=None):
    """x [M, K] -> (codes uint8 [M, kp], scale bytes uint8 [M, nb], row scales fp32 [M] or None)."""
    g = 16 if fmt == F.FMT_NVFP4 else 32
    m, k = x.shape
    kp = -(-k // 32) * 32
    v = torch.zeros(m, kp, dtype=torch.float64)
    v[:, :k] = x.cpu().double()
    b = v.view(m, kp // g, g)
    fin = torch.isfinite(b).all(-1)
    amax = torch.where(fin, b.abs().amax(-1), torch.zeros((), dtype=torch.float64))
    t = None
    if fmt == F.FMT_NVFP4:
        if ts is None:
            t = (amax.amax(1) / 2688).float().clamp_min(2.0 ** -126)
            d = t.double()[:, None]
        else:
            d = ts.cpu().double().view(1, 1)
        sb = nearest((amax / (6 * d)).clamp_max(448.0), E4M3)
        s = E4M3[sb] * d
        sb = torch.where(fin, sb, torch.full_like(sb, 0x7F))
    else:
        mant, e = torch.frexp(amax.clamp_min(6 * 2.0 ** -126))       # amax = mant 2^e, mant in [0.5, 1)
        p = torch.where(mant <= 0.75, e - 3, e - 2)                  # mant 2^e <= 6 2^p  iff  mant / 0.75 <= 2^(p + 3 - e)
        s = torch.ldexp(torch.ones_like(amax), p)
        sb = torch.where(fin, p + 127, torch.full_like(p, 255)).long()
    q = torch.where((s > 0)[..., None], b.abs() / torch.where(s > 0, s, 1.0)[..., None], torch.zeros_like(b))
    mag = nearest(q.nan_to_num(0.0, 0.0).clamp_max(6.0), MAGS)
    c = mag + 8 * (torch.signbit(b) & (s > 0)[..., None]).long()
    c = torch.where(fin[..., None], c, torch.zeros_like(c))
    return c.view(m, kp).to(torch.uint8), sb.to(torch.uint8), t


def values(codes, sb, fmt, ts=None):
    """fp64 values [M, kp] of codes and scale bytes; ts fp32 [M] or [1]."""
    g = 16 if fmt == F.FMT_NVFP4 else 32
    mag = MAGS[(codes & 7).long()]
    v = torch.where(codes >= 8, -mag, mag)
    if fmt == F.FMT_NVFP4:
        s = torch.cat([E4M3, torch.tensor([math.nan], dtype=torch.float64)])[(sb & 0x7F).long()]
        if ts is not None:
            s = s * ts.cpu().double().view(-1, 1)
    else:
        s = torch.where(sb == 255, math.nan, torch.pow(2.0, sb.double() - 127))
    return (v.view(v.shape[0], -1, g) * s[..., None]).view(v.shape)


def unpack(packed):
    p = packed.cpu()
    return torch.stack([p & 15, p >> 4], -1).flatten(-2)


def weights(fmt, n, k, seed, mats=1, halves=1):
    """Random canonical weights on the CPU: codes [mats, n, k/2], scale bytes, ts [mats, halves] or None, and
    their fp64 values [mats, n, k]."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (mats, n, k // 2), generator=g, dtype=torch.uint8)
    nb = k // (16 if fmt == F.FMT_NVFP4 else 32)
    lo, hi = (0x20, 0x70) if fmt == F.FMT_NVFP4 else (116, 124)
    s = torch.randint(lo, hi, (mats, n, nb), generator=g, dtype=torch.uint8)
    ts = 0.01 * (1 + torch.rand(mats, halves, generator=g)) if fmt == F.FMT_NVFP4 else None
    v = []
    for e in range(mats):
        w = values(unpack(codes[e]), s[e], fmt)
        if ts is not None:
            w = (w.view(halves, n // halves, k) * ts[e].double().view(halves, 1, 1)).view(n, k)
        v.append(w)
    return codes, s, ts, torch.stack(v)


def route(logits, k, bias=None, score="sigmoid", n_group=1, topk_group=1, group_score="max", renormalize=True, scale=1.0):
    """(weights fp64 [T, k], ids [T, k]) of CPU logits [T, E], token by token."""
    low = torch.finfo(logits.dtype).min
    l = logits.double()
    masked = ~(l > low)
    l = torch.where(masked, -math.inf, l.clamp_max(torch.finfo(torch.float32).max))
    if score == "softmax":
        mx = torch.where(masked.all(1, keepdim=True), 0.0, l.amax(1, keepdim=True))
        s = torch.exp(l - mx)
        s = s / s.sum(1, keepdim=True).clamp_min(1e-300)
    elif score == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        s = torch.sqrt(l.clamp_min(0) + torch.log1p(torch.exp(-l.abs())))
    s = torch.where(masked, 0.0, s)
    pick = l if bias is None else torch.where(masked, -math.inf, s + bias.double())
    by_group = pick if bias is not None or group_score == "max" else torch.where(masked, -math.inf, s)
    t, e = l.shape
    size = e // n_group
    ids = torch.empty(t, k, dtype=torch.int64)
    w = torch.zeros(t, k, dtype=torch.float64)
    for i in range(t):
        allowed = list(range(e))
        if n_group > 1:
            gs = []
            for g in range(n_group):
                b = sorted(by_group[i, g * size:(g + 1) * size].tolist(), reverse=True)[:2 if group_score == "top2" else 1]
                gs.append(-math.inf if b[0] == -math.inf else sum(x for x in b if x > -math.inf))
            kept = sorted(range(n_group), key=lambda g: (-gs[g], g))[:topk_group]
            allowed = [g * size + j for g in sorted(kept) for j in range(size)]
        p = pick[i].tolist()
        best = sorted(allowed, key=lambda j: (-p[j], j))[:k]
        ids[i] = torch.tensor(best)
        c = s[i, ids[i]]
        if renormalize:
            c = c / c.sum() if c.sum() > 0 else torch.zeros_like(c)
        w[i] = c * scale
    return w, ids


def order(ids, e):
    """(offsets, tokens, places) of ids [T, k] as lists."""
    t, k = ids.shape
    flat = ids.reshape(-1).tolist()
    lists = [[p for p in range(t * k) if flat[p] == x] for x in range(e)]
    offsets, tokens, places = [0], [], [-1] * (t * k)
    for x in lists:
        for p in x:
            places[p] = len(tokens)
            tokens.append(p // k)
        offsets.append(len(tokens))
    return offsets, tokens + [-1] * (t * k - len(tokens)), places
