"""The 8-bit block cache and beam search in 64 bits, row by row, as the header defines them: what the kernels are held to."""
import math

import torch

BLOCK, LOW, HIGH = 32, -40, 40
F64 = torch.float64


def exponent(top: float) -> int:
    """The least e with top <= 448 * 2^e, within the cache's range."""
    if top == 0:
        return LOW
    e = math.frexp(top)[1] - 9
    while top > math.ldexp(448, e):
        e += 1
    return min(max(e, LOW), HIGH)


def e4m3(y: torch.Tensor) -> torch.Tensor:
    """The e4m3 number next to y, ties to even, saturated; NaN counts as 0."""
    y = torch.nan_to_num(y.double(), nan=0.0, posinf=448.0, neginf=-448.0).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(y / step) * step


def value_of(codes: torch.Tensor) -> torch.Tensor:
    code = codes.to(torch.int64)
    power, part = (code >> 3) & 15, (code & 7).double()
    size = torch.where(power == 0, part * 2.0**-9, (1 + part / 8) * torch.exp2(power.double() - 7))
    return torch.where(code >= 128, -size, size)


def held(codes, exps):
    """Codes [..., rows, dim], scale bytes [..., rows / 32] -> what they stand for, in 64 bits."""
    return value_of(codes) * torch.exp2(exps.double() - 127).repeat_interleave(BLOCK, -1)[..., None]


def finite_top(x: torch.Tensor) -> float:
    x = x.double().abs()
    return float(torch.where(torch.isfinite(x), x, 0).max()) if x.numel() else 0.0


def append(values, exps, x, r0, n):
    """values [ctx, dim] (64 bits), exps [blocks] (ints), x [tokens, dim]: rows r0 .. r0 + n - 1, in place."""
    ctx = values.shape[0]
    if r0 < 0 or r0 >= ctx or n <= 0:
        return
    end = min(r0 + min(n, x.shape[0]), ctx)
    for blk in range(r0 // BLOCK, (end - 1) // BLOCK + 1):
        lo, hi = max(blk * BLOCK, r0), min((blk + 1) * BLOCK, end)
        new = x[lo - r0 : hi - r0]
        e = exponent(finite_top(new))
        if blk * BLOCK < r0:
            if e <= exps[blk]:
                e = exps[blk]
            else:
                old = values[blk * BLOCK : r0]
                values[blk * BLOCK : r0] = e4m3(old * 2.0**-e) * 2.0**e
        values[lo:hi] = e4m3(new.double() * 2.0**-e) * 2.0**e
        exps[blk] = e


def limits(kv_len, pos0, tokens, prefix):
    p = pos0 + torch.arange(tokens)
    n = torch.where(p < prefix, torch.clamp(p + 1, min=prefix), p + 1)
    return torch.where(p < 0, 0, torch.clamp(n, max=kv_len))


def attention(q, k, v, kv_len, pos0, prefix, scale):
    """q [tokens, heads, dim], k, v [kv_heads, ctx, dim] -> (o, weight of every row [kv_heads, ctx], sum of p |v| [tokens, heads, dim],
    largest |score|, largest sum of |q k|): 64 bits."""
    tokens, heads, dim = q.shape
    kv_heads, ctx = k.shape[:2]
    group = heads // kv_heads
    lim = limits(kv_len, pos0, tokens, prefix)
    o = torch.zeros(tokens, heads, dim, dtype=F64)
    size = torch.zeros(tokens, heads, dim, dtype=F64)
    w = torch.zeros(kv_heads, ctx, dtype=F64)
    most = mass = 0.0
    n = int(kv_len)
    if n == 0:
        return o, w, size, most, mass
    see = torch.arange(n)[None] < lim[:, None]
    for h in range(heads):
        kk, vv = k[h // group, :n].double(), v[h // group, :n].double()
        t = q[:, h].double() @ kk.T * scale
        p = torch.softmax(t.masked_fill(~see, -math.inf), -1)
        p = torch.where(see, p, 0.0)
        o[:, h], size[:, h] = p @ vv, p @ vv.abs()
        w[h // group, :n] += p.sum(0)
        if bool(see.any()):
            most = max(most, float(t[see].abs().max()))
            mass = max(mass, float((q[:, h].double().abs() @ kk.abs().T * scale).max()))
    return o, w, size, most, mass


def attention_tolerance(o, size, most, mass, dim, kv_len, v_top):
    """What the kernel's roundings may come to.  Scores: `dim` products summed in fp32 (dim * 2^-24 of the sum of magnitudes) and the exponent's
    rounding (2^-24 of its size, taken in units of log2): a relative error d of every weight, twice in the quotient.  A weight enters the product
    with the values as fp16: 2^-11 relative, or 2^-25 of the largest where it is subnormal there.  fp32 sums over the keys: kv_len * 2^-24 at most.
    The output is rounded to bf16: 2^-8."""
    d = dim * 2.0**-24 * mass + (most + 50) * 1.45 * 2.0**-23 + 2.0**-21
    return o.abs() * 2.0**-8 + size * (2.0**-11 + 2 * d + kv_len * 2.0**-23) * (1 + 2.0**-8) + kv_len * 2.0**-25 * v_top


def weights_tolerance(w, most, mass, dim, columns):
    d = dim * 2.0**-24 * mass + (most + 50) * 1.45 * 2.0**-23 + 2.0**-21
    return w * (2 * d + columns * 2.0**-24 + 2.0**-20) + 1e-12


def kept_rows(w, n, keep, first, recent):
    """Row numbers that stay, of weights [n] -- plain sorting, ties to the lower row, NaN least."""
    if n <= keep:
        return list(range(n))
    forced = set(range(first)) | set(range(max(0, n - recent), n))
    key = lambda j: -math.inf if math.isnan(w[j]) else w[j]  # noqa: E731
    rest = sorted((j for j in range(n) if j not in forced), key=lambda j: (-key(j), math.isnan(w[j]), j))
    return sorted(list(forced) + rest[: keep - len(forced)])


def beams(logits, scores, ended, end_id, suppress_id, rank_weight):
    """One input: logits [beams, vocab], scores [beams] -> lists of (token, parent, score, ended)."""
    k, v = logits.shape
    cand = []
    for i in range(k):
        s = float(scores[i])
        if not s > -math.inf:
            continue
        wt = float(rank_weight[i]) if rank_weight is not None else 1.0
        if ended is not None and int(ended[i]):
            cand.append((s * wt, i, 0.0, end_id, s, 1))
            continue
        x = logits[i].double().clone()
        x[torch.isnan(x)] = -math.inf
        x = torch.clamp(x, max=3.4028234663852886e38)
        if 0 <= suppress_id < v:
            x[suppress_id] = -math.inf
        if not bool((x > -math.inf).any()):
            continue
        m = x.max()
        lse = m + torch.log(torch.exp(x - m).sum())
        best = torch.sort(x, descending=True, stable=True)
        for t, l in zip(best.indices[: k].tolist(), best.values[: k].tolist()):
            total = s + (l - float(lse))
            if total > -math.inf:
                cand.append((total * wt, i, l, t, total, int(t == end_id)))
    cand.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
    out = [(c[3], c[1], c[4], c[5]) for c in cand[:k]]
    return out + [(end_id, i, -math.inf, 1) for i in range(len(out), k)]
