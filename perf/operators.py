"""The operators of long and many-beamed answers over an 8-bit cache, as cases that can be timed and compared.

A block cache holds keys and values as e4m3 numbers with one power-of-two scale for each block of 32 tokens and head
(``moondream_amd.block_cache.BlockCache``); next to it stands the choice among beams (``moondream_amd.beams``):

  append     new tokens' keys and values (a decode step's, or a ragged batch of prompts) into the cache; the rows are read back
  attention  queries over the cache: single tokens, a few, or prompts; optionally the weight that each cached token got
  evict      the cached tokens of least accumulated weight leave, the others move together into a smaller cache; read back
  beam       the best continuations of every input's beams, then the beams' states behind their parents

The plain forms are elementary torch operations in 32 bits; what decides a choice (beams' totals) is in 64.
"""
import math
import random

import torch

own = False

BLOCK = 32
LOW, HIGH = -40, 40  # exponents of a block's scale
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
DEV = "cuda"


# ----------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of the 2B model's answers in lockstep: 64 sequences of an image (730 tokens), a question and some answer
        dict(name="append-step", kind="append", batch=64, kv_heads=32, heads=32, dim=64, ctx=1024, new=1, ragged=False, start=770),
        # questions and long texts of eight conversations behind their images, every one of another length
        dict(name="append-prompts", kind="append", batch=8, kv_heads=32, heads=32, dim=64, ctx=4096, new=2000, ragged=True, start=730),
        # one sequence's decode step behind an image: latency is all that counts
        dict(name="attention-one", kind="attention", batch=1, heads=32, kv_heads=32, dim=64, new=1, len=778, ragged=False, prefix=0, weights=False),
        # the lockstep decode step of 64 answers
        dict(name="attention-answers", kind="attention", batch=64, heads=32, kv_heads=32, dim=64, new=1, len=1003, ragged=True, prefix=0, weights=False),
        # long conversations on shared heads, the weights of every cached token kept for the eviction
        dict(name="attention-long", kind="attention", batch=8, heads=32, kv_heads=8, dim=128, new=1, len=32749, ragged=True, prefix=0, weights=True),
        # eight images and their questions read at once: the image's 730 tokens see one another
        dict(name="attention-images", kind="attention", batch=8, heads=32, kv_heads=32, dim=64, new=767, len=767, ragged=False, prefix=730, weights=False),
        # a long prompt's second portion on shared heads, with the weights that its tokens give
        dict(name="attention-portion", kind="attention", batch=2, heads=32, kv_heads=8, dim=128, new=2048, len=6101, ragged=True, prefix=0, weights=True),
        # a conversation behind an image is cut to 512 tokens a head
        dict(name="evict-one", kind="evict", batch=1, kv_heads=32, dim=64, len=801, ragged=False, keep=512, first=4, recent=64),
        # long conversations are cut to an eighth
        dict(name="evict-long", kind="evict", batch=8, kv_heads=8, dim=128, len=32749, ragged=True, keep=4096, first=4, recent=256),
        # an answer of four beams: the 2B model's vocabulary and its cache of 24 layers, 30 tokens into the answer
        dict(name="beam-one", kind="beam", batch=1, beams=4, vocab=51200, f32=False, layers=24, heads=32, rows=32, dim=64, state="bf16"),
        # sixteen images' answers of four beams, 60 tokens into the answers
        dict(name="beam-images", kind="beam", batch=16, beams=4, vocab=51200, f32=False, layers=24, heads=32, rows=64, dim=64, state="bf16"),
        # many beams of a layered model: fp32 logits of a large vocabulary, the states of its retention layers
        dict(name="beam-states", kind="beam", batch=4, beams=16, vocab=131075, f32=True, layers=12, heads=16, rows=64, dim=64, state="f32"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "evict", "beam"])
    if kind == "beam":
        while True:
            state = rng.choice(["bf16", "f32"])
            c = dict(kind=kind, batch=_spread(rng, 1, 32), beams=rng.choice([2, 3, 4, 5, 8, 16]), vocab=_spread(rng, 1000, 140000), f32=rng.random() < 0.5,
                     layers=rng.choice([2, 12, 24]), heads=rng.choice([8, 16, 32]), rows=rng.choice([16, 32, 33, 64, 100]) if state == "bf16" else 64, dim=64, state=state)
            if c["batch"] * c["beams"] * c["vocab"] <= 8 << 20 and work(c)["bytes"] <= 1.5e9:
                return c
    dim, group = rng.choice([64, 128]), rng.choice([1, 1, 2, 4, 5, 8])
    while True:
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
        batch = _spread(rng, 1, 64)
        if kind == "append":
            new = rng.choice([1, _spread(rng, 1, 2048)])
            start = rng.randrange(0, 2000)
            c = dict(kind=kind, batch=batch, kv_heads=kv_heads, heads=kv_heads * group, dim=dim, ctx=4096, new=new, ragged=rng.random() < 0.5, start=start)
            if batch * kv_heads * dim <= 8 * 32 * 64 * (8 if new == 1 else 1):
                return c
        if kind == "attention":
            new = rng.choice([1, 1, rng.randrange(2, 9), _spread(rng, 9, 2048)])
            length = max(new, _spread(rng, 1, 32768))
            c = dict(kind=kind, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, new=new, len=length, ragged=rng.random() < 0.6,
                     prefix=rng.choice([0, 0, min(length, 730)]), weights=rng.random() < 0.4)
            if work(c)["flops"] <= 1.5e11 and batch * kv_heads * length * dim <= 8 * 8 * 32768 * 128 and batch * c["heads"] * new * length <= 1 << 30:
                return c
        if kind == "evict":
            length = _spread(rng, 40, 32768)
            keep = rng.randrange(33, length + 33)
            c = dict(kind=kind, batch=batch, kv_heads=kv_heads, dim=dim, len=length, ragged=rng.random() < 0.5, keep=keep, first=rng.choice([0, 1, 4]), recent=rng.choice([0, 7, 28]))
            if batch * kv_heads * length * dim <= 8 * 8 * 32768 * 128 and batch * kv_heads * keep * dim <= 8 * 8 * 4096 * 128:
                return c


def _lengths(c):
    """Of a ragged batch: from half the longest to the longest, spread evenly; a decode step's and a prompt's alike."""
    b, n = c["batch"], c["len"]
    least = max(c.get("new", 1), (n + 1) // 2)
    return [n - (n - least) * i // max(1, b - 1) for i in range(b)] if c["ragged"] else [n] * b


def _new_rows(c):
    return [c["new"] - c["new"] // 2 * i // max(1, c["batch"] - 1) for i in range(c["batch"])] if c["ragged"] else [c["new"]] * c["batch"]


def work(c):
    if c["kind"] == "append":  # bf16 rows in; codes out, in again, values out
        rows = sum(_new_rows(c)) * c["kv_heads"] * c["dim"] * 2
        return {"bytes": rows * (2 + 1 + 1 + 2), "flops": 0}
    if c["kind"] == "attention":
        pairs = bytes_ = 0
        for n in _lengths(c):
            first = n - c["new"]
            pairs += sum(max(p + 1, min(n, c["prefix"]) if p < c["prefix"] else 0) for p in range(first, n)) * c["heads"]
            bytes_ += n * c["kv_heads"] * (2 * c["dim"] + 2 / BLOCK) + c["new"] * c["heads"] * c["dim"] * 4 + (n * c["kv_heads"] * 4 if c["weights"] else 0)
        return {"bytes": bytes_, "flops": pairs * c["dim"] * 4}
    if c["kind"] == "evict":  # weights in; kept rows' codes in and out, in again, values out
        lens = _lengths(c)
        kept = sum(min(n, c["keep"]) for n in lens) * c["kv_heads"]
        return {"bytes": sum(lens) * c["kv_heads"] * 4 + kept * (c["dim"] * 2 * (1 + 1 + 1 + 2) + 8), "flops": 0}
    slots = c["batch"] * c["beams"]
    state = c["layers"] * slots * c["heads"] * c["rows"] * c["dim"] * (4 if c["state"] == "bf16" else 4)  # bf16: keys and values
    return {"bytes": slots * c["vocab"] * (4 if c["f32"] else 2) + 2 * state, "flops": 0}


# ------------------------------------------------------------------------------------------------------- numbers in the cache
def _quantise(x):
    """Blocks [..., 32, dim] in fp32 -> (e4m3 codes as bytes, exponents [...]): the least power of two that keeps a block within 448."""
    top = x.abs().amax((-1, -2))
    part, power = torch.frexp(top)
    e = (power - 9 + (part > 0.875).to(I32)).clamp(LOW, HIGH)
    e = torch.where(top > 0, e, torch.full_like(e, LOW))
    y = torch.ldexp(x, -e[..., None, None]).clamp(-448, 448)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), e


def _values(codes, exps):
    """Codes [..., rows, dim] and scale bytes [..., rows / 32] -> fp32."""
    scale = torch.ldexp(torch.ones((), dtype=F32, device=codes.device), exps.to(I32) - 127)
    return codes.view(torch.float8_e4m3fn).to(F32) * scale.repeat_interleave(BLOCK, -1)[..., None]


def _filled(g, slots, heads, ctx, dim, loud):
    """A cache as real ones are: some channels many times larger than others, another size in every head."""
    codes, exps = [], []
    size = torch.exp2(torch.randn(heads, 1, 1, device=DEV, generator=g)) * torch.where(torch.rand(heads, 1, dim, device=DEV, generator=g) < 0.05, loud, 1.0)
    for _ in range(slots):  # a slot at a time: 32-bit values of the whole cache need not fit
        c, e = _quantise((torch.randn(heads, ctx, dim, device=DEV, generator=g) * size).view(heads, ctx // BLOCK, BLOCK, dim))
        codes.append(c.view(heads, ctx, dim))
        exps.append((e + 127).to(torch.uint8))
    return torch.stack(codes), torch.stack(exps)


def _up(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(c=c)
    if c["kind"] == "append":
        b, n, h, kh, d = c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"]
        s["k"], s["k_exp"] = _filled(g, b, kh, c["ctx"], d, 1.0)
        s["v"], s["v_exp"] = s["k"].clone(), s["k_exp"].clone()
        # the projection's rows: queries, keys and values of a token one after another
        s["qkv"] = (torch.randn(b, n, (h + 2 * kh) * d, device=DEV, generator=g) * torch.exp2(torch.randn(b, n, 1, device=DEV, generator=g))).to(BF16)
        counts = _new_rows(c)
        s["rows"] = max(counts)
        starts = [c["start"] - min(c["start"], 7 * i % 200) for i in range(b)] if c["ragged"] or n == 1 else [c["start"]] * b
        s["row0"] = torch.tensor(starts, dtype=I32, device=DEV)
        s["new"] = torch.tensor(counts, dtype=I32, device=DEV)
        s["read0"] = torch.div(s["row0"], BLOCK, rounding_mode="floor").to(I32) * BLOCK  # from the start of the first block written
        s["len"] = s["row0"] + s["new"]
        s["back"] = _up(n + BLOCK - 1)
    elif c["kind"] == "attention":
        b, n, h, kh, d = c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"]
        ctx = _up(c["len"])
        s["k"], s["k_exp"] = _filled(g, b, kh, ctx, d, 4.0)
        s["v"], s["v_exp"] = _filled(g, b, kh, ctx, d, 1.0)
        # scores of a few units: some tokens get most of the weight
        s["q"] = (torch.randn(b, n, h, d, device=DEV, generator=g) * 0.7).to(BF16)
        s["len"] = torch.tensor(_lengths(c), dtype=I32, device=DEV)
        s["longest"] = c["len"]
        s["weights"] = torch.zeros(b, kh, ctx, device=DEV) if c["weights"] else None
    elif c["kind"] == "evict":
        b, kh, d = c["batch"], c["kv_heads"], c["dim"]
        ctx, room = _up(c["len"]), _up(c["keep"])
        s["k"], s["k_exp"] = _filled(g, b, kh, ctx, d, 4.0)
        s["v"], s["v_exp"] = _filled(g, b, kh, ctx, d, 1.0)
        s["weights"] = torch.exp(2 * torch.randn(b, kh, ctx, device=DEV, generator=g))
        s["len"] = torch.tensor(_lengths(c), dtype=I32, device=DEV)
        s["read0"] = torch.zeros(b, dtype=I32, device=DEV)
        for x in ("k", "v"):
            s["into_" + x] = torch.zeros(b, kh, room, d, dtype=torch.uint8, device=DEV)
            s["into_" + x + "_exp"] = torch.full((b, kh, room // BLOCK), 127, dtype=torch.uint8, device=DEV)
        s["into_weights"] = torch.zeros(b, kh, room, device=DEV)
    else:
        b, k, v = c["batch"], c["beams"], c["vocab"]
        s["logits"] = (torch.randn(b * k, v, device=DEV, generator=g) * 2).to(F32 if c["f32"] else BF16)
        s["scores"] = -torch.rand(b, k, device=DEV, generator=g) * 12
        s["ended"] = (torch.rand(b, k, device=DEV, generator=g) < 0.15).to(I32)
        if c["state"] == "bf16":
            shape = (c["layers"], b * k, c["heads"], c["rows"], c["dim"])
            s["states"] = [torch.randn(shape, device=DEV, generator=g, dtype=BF16) for _ in range(2)]
        else:
            s["states"] = [torch.randn((c["layers"], b * k, c["heads"], c["rows"], c["dim"]), device=DEV, generator=g)]
        s["into"] = [torch.zeros_like(x) for x in s["states"]]
    if own:
        from moondream_amd.block_cache import BlockCache

        if "k_exp" in s:
            s["cache"] = BlockCache.of(s["k"], s["v"], s["k_exp"], s["v_exp"])
        if "into_k" in s:
            s["small"] = BlockCache.of(s["into_k"], s["into_v"], s["into_k_exp"], s["into_v_exp"])
    return s


# ------------------------------------------------------------------------------------------------------------ the plain forms
def _plain_append_one(x, codes, exps, row0, new, rows):
    """x [b, n, heads, dim] behind row0 of codes / exps, in place; the rows of the touched blocks, zeros behind the last."""
    b, n, heads, dim = x.shape
    nb = (rows + 2 * BLOCK - 2) // BLOCK
    first = torch.div(row0, BLOCK, rounding_mode="floor")
    blocks = (first[:, None] + torch.arange(nb, device=DEV)).long()
    fits = blocks < exps.shape[2]
    at = blocks.clamp(max=exps.shape[2] - 1)
    row = blocks[:, :, None] * BLOCK + torch.arange(BLOCK, device=DEV)  # [b, nb, 32]
    seq = torch.arange(b, device=DEV)
    fresh = ((row >= row0[:, None, None]) & (row < (row0 + new)[:, None, None]))[..., None, None]
    old = (row < row0[:, None, None])[..., None, None]
    taken = x.float()[seq[:, None, None], (row - row0[:, None, None]).clamp(0, n - 1)]  # [b, nb, 32, heads, dim]
    taken = torch.where(fresh, taken, 0).permute(0, 3, 1, 2, 4)
    old_codes = codes.view(b, heads, -1, BLOCK, dim)[seq[:, None], :, at].transpose(1, 2)  # [b, heads, nb, 32, dim]
    old_e = exps[seq[:, None], :, at].transpose(1, 2).to(I32) - 127
    was = torch.where(old.permute(0, 3, 1, 2, 4), torch.ldexp(old_codes.view(torch.float8_e4m3fn).float(), old_e[..., None, None]), 0)
    _, e = _quantise(taken)
    e = torch.where(old.any(2)[..., 0, 0][:, None], torch.maximum(e, old_e), e)
    got = torch.ldexp(taken + was, -e[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = (fresh | old).permute(0, 3, 1, 2, 4)
    got = torch.where(keep, got, old_codes)
    some = (fits & fresh.any(2)[..., 0, 0])
    where = torch.nonzero(some)
    codes.view(b, heads, -1, BLOCK, dim)[where[:, 0], :, blocks[some]] = got.transpose(1, 2)[some]
    exps[where[:, 0], :, blocks[some]] = (e.transpose(1, 2)[some] + 127).to(torch.uint8)
    back = torch.ldexp(torch.where(keep, got, 0).view(torch.float8_e4m3fn).float(), e[..., None, None])
    return back.reshape(b, heads, nb * BLOCK, dim).to(BF16)


def _plain_append(s):
    c = s["c"]
    k, v = _keys_values(s)
    got = [_plain_append_one(x, s[y], s[y + "_exp"], s["row0"], s["new"], c["new"]) for x, y in ((k, "k"), (v, "v"))]
    rows = torch.arange(s["back"], device=DEV)
    live = ((s["read0"][:, None] + rows) < s["len"][:, None])[:, None, :, None]
    return [torch.where(live, x[:, :, : s["back"]], 0) for x in got]


def _keys_values(s):
    c = s["c"]
    h, kh, d = c["heads"], c["kv_heads"], c["dim"]
    rows = s["qkv"].view(c["batch"], c["new"], h + 2 * kh, d)
    return rows[:, :, h : h + kh], rows[:, :, h + kh :]


def _visible(s, ctx):
    """[b, new, ctx]: key j is seen from position p if j <= p, or if both lie in the prefix."""
    c = s["c"]
    p = (s["len"] - c["new"])[:, None] + torch.arange(c["new"], device=DEV)
    limit = torch.where(p < c["prefix"], torch.clamp(p + 1, min=c["prefix"]), p + 1)
    limit = torch.minimum(limit, s["len"][:, None])
    return torch.arange(ctx, device=DEV) < limit[..., None]


def _plain_attention(s):
    c = s["c"]
    b, n, h, kh, d = c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"]
    ctx = s["k"].shape[2]
    k, v = _values(s["k"], s["k_exp"]), _values(s["v"], s["v_exp"])
    q = s["q"].float().view(b, n, kh, h // kh, d).permute(0, 2, 3, 1, 4).reshape(b, kh, h // kh * n, d)
    see = _visible(s, ctx).repeat(1, h // kh, 1)[:, None]
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).masked_fill_(~see, -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p, v).view(b, kh, h // kh, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(BF16)
    return [o, p.sum(2)] if c["weights"] else [o]


def _plain_evict(s):
    c = s["c"]
    b, kh, d, keep = c["batch"], c["kv_heads"], c["dim"], c["keep"]
    ctx, room = s["k"].shape[2], s["into_k"].shape[2]
    j, n = torch.arange(ctx, device=DEV), s["len"][:, None]
    rank = torch.where(((j < c["first"]) | (j >= n - c["recent"]))[:, None], math.inf, s["weights"])
    rank = torch.where((j < n)[:, None], rank, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.nn.functional.pad(best, (0, max(0, room - best.shape[-1])), value=ctx)
    live = torch.arange(room, device=DEV) < torch.clamp(n, max=keep)
    best = torch.sort(torch.where(live[:, None], best, ctx), -1).values  # in the order of their rows; nothing behind the last
    at = best.clamp(max=ctx - 1)
    got = []
    for x in ("k", "v"):
        codes = torch.gather(s[x], 2, at[..., None].expand(-1, -1, -1, d)).view(torch.float8_e4m3fn).float()
        rows = torch.ldexp(codes, torch.gather(s[x + "_exp"], 2, at // BLOCK).to(I32)[..., None] - 127)
        rows = torch.where(live[:, None, :, None], rows, 0).view(b, kh, room // BLOCK, BLOCK, d)
        codes, e = _quantise(rows)
        s["into_" + x].copy_(codes.view(b, kh, room, d))
        s["into_" + x + "_exp"].copy_((e + 127).to(torch.uint8))
        got.append(_values(s["into_" + x], s["into_" + x + "_exp"]).to(BF16))
    kept = torch.where(live[:, None, :keep], best[..., :keep], -1).to(I32)
    s["into_weights"].copy_(torch.where(live[:, None], torch.gather(s["weights"], 2, at), 0))
    return [kept, torch.clamp(s["len"], max=keep), s["into_weights"][..., :keep], *got]


END = 0


def _plain_beam(s):
    c = s["c"]
    b, k, v = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - top - (x - top).exp().sum(-1, keepdim=True).log() + s["scores"].double().view(-1, 1)
    only = torch.full_like(x, -math.inf)  # an ended beam goes on as it is
    only[:, END] = s["scores"].double().view(-1)
    x = torch.where(s["ended"].view(-1, 1) != 0, only, x).view(b, k * v)
    total, at = torch.sort(x, dim=-1, descending=True, stable=True)
    total, at = total[:, :k], at[:, :k]
    parents = torch.div(at, v, rounding_mode="floor")
    tokens = at - parents * v
    ended = ((torch.gather(s["ended"], 1, parents) != 0) | (tokens == END)).to(I32)
    slots = (parents + torch.arange(b, device=DEV)[:, None] * k).view(-1)
    for old, new in zip(s["states"], s["into"]):
        torch.index_select(old, 1, slots, out=new)
    return [tokens.to(I32), parents.to(I32), total.float(), ended, *s["into"]]


def run(state):
    s, kind = state, state["c"]["kind"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict, "beam": _plain_beam}[kind](s)
    c = s["c"]
    if kind == "append":
        k, v = _keys_values(s)
        s["cache"].append(k, v, s["row0"], new=s["new"])
        return list(s["cache"].read(s["read0"], s["back"], kv_len=s["len"]))
    if kind == "attention":
        o = s["cache"].attention(s["q"], s["len"], prefix_len=c["prefix"], max_len=s["longest"], weights=s["weights"], decay=0.0)
        return [o, s["weights"]] if c["weights"] else [o]
    if kind == "evict":
        kept, length = s["cache"].evict(s["weights"], s["len"], c["keep"], first=c["first"], recent=c["recent"], into=s["small"], into_weights=s["into_weights"])
        return [kept, length, s["into_weights"][..., : c["keep"]], *s["small"].read(s["read0"], s["into_k"].shape[2], kv_len=length)]
    from moondream_amd.beams import reorder_states, select_beams

    tokens, parents, scores, ended = select_beams(s["logits"], s["scores"], ended=s["ended"], end_id=END)
    reorder_states(s["states"], parents, into=s["into"], slot_dim=1)
    return [tokens, parents, scores, ended, *s["into"]]


# ------------------------------------------------------------------------------------------------------- in 64 bits, by itself
def _e4m3(y):
    """The e4m3 number next to y (|y| <= 448), ties to even: steps of an eighth of the power of two below, of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(y / step) * step


def _scale_of(top):
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448))
    e = torch.where(torch.exp2(e) * 448 < top, e + 1, torch.where(torch.exp2(e - 1) * 448 >= top, e - 1, e))
    return torch.exp2(e.clamp(LOW, HIGH))


def _held(codes, exps):
    """What a byte stands for, from its fields: sign, four bits of exponent, three of fraction."""
    code = codes.to(torch.int64)
    power, part = (code >> 3) & 15, (code & 7).double()
    size = torch.where(power == 0, part * 2.0**-9, (1 + part / 8) * torch.exp2(power.double() - 7))
    value = torch.where(code >= 128, -size, size)
    return value * torch.exp2(exps.double() - 127).repeat_interleave(BLOCK, -1)[..., None]


def exact(case, seed):
    c = case
    s = prepare(dict(c), seed)
    if c["kind"] == "attention":
        b, n, h, kh, d = c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"]
        o = torch.zeros(b, n, h, d, dtype=F64, device=DEV)
        w = torch.zeros(b, kh, s["k"].shape[2], dtype=F64, device=DEV)
        for i, length in enumerate(_lengths(c)):
            k, v = (_held(s[x][i], s[x + "_exp"][i])[:, :length] for x in ("k", "v"))
            at = torch.arange(length - n, length, device=DEV)[:, None]
            key = torch.arange(length, device=DEV)
            hidden = ~((key <= at) | ((at < c["prefix"]) & (key < c["prefix"])))
            for j in range(h):
                t = (s["q"][i, :, j].double() @ k[j // (h // kh)].T) / math.sqrt(d)
                p = torch.softmax(t.masked_fill(hidden, -math.inf), -1)
                o[i, :, j] = p @ v[j // (h // kh)]
                w[i, j // (h // kh), :length] += p.sum(0)
        return [o, w] if c["weights"] else [o]
    if c["kind"] == "append":
        got = []
        for x, name in zip(_keys_values(s), ("k", "v")):
            out = torch.zeros(c["batch"], c["kv_heads"], s["back"], c["dim"], dtype=F64, device=DEV)
            for i in range(c["batch"]):
                r0, m, z = int(s["row0"][i]), int(s["new"][i]), int(s["read0"][i])
                before = _held(s[name][i, :, z : z + BLOCK], s[name + "_exp"][i, :, z // BLOCK : z // BLOCK + 1])[:, : r0 - z]
                rows = torch.cat([before, x[i, :m].double().transpose(0, 1)], 1)
                rows = torch.nn.functional.pad(rows, (0, 0, 0, -rows.shape[1] % BLOCK)).view(c["kv_heads"], -1, BLOCK, c["dim"])
                fresh = rows.clone()
                fresh[:, 0, : r0 - z] = 0
                scale = _scale_of(fresh.abs().amax((-1, -2)))
                if r0 > z:
                    scale[:, 0] = torch.maximum(scale[:, 0], torch.exp2(s[name + "_exp"][i, :, z // BLOCK].double() - 127))
                rows = (_e4m3((rows / scale[..., None, None]).clamp(-448, 448)) * scale[..., None, None]).flatten(1, 2)
                out[i, :, : r0 - z + m] = rows[:, : r0 - z + m]
            got.append(out)
        return got
    if c["kind"] == "evict":
        keep, room = c["keep"], s["into_k"].shape[2]
        out = [torch.zeros(c["batch"], c["kv_heads"], room, c["dim"], dtype=F64, device=DEV) for _ in range(2)]
        left = torch.zeros(c["batch"], c["kv_heads"], keep, dtype=F64, device=DEV)
        for i, n in enumerate(_lengths(c)):
            w = s["weights"][i, :, :n].double()
            w[:, : c["first"]] = math.inf
            w[:, n - c["recent"] :] = math.inf
            m = min(n, keep)
            at = torch.argsort(-w, dim=-1, stable=True)[:, :m].sort(-1).values
            left[i, :, :m] = torch.gather(s["weights"][i], 1, at)
            for x, y in zip(("k", "v"), out):
                rows = torch.gather(_held(s[x][i], s[x + "_exp"][i]), 1, at[..., None].expand(-1, -1, c["dim"]))
                rows = torch.nn.functional.pad(rows, (0, 0, 0, -m % BLOCK)).view(c["kv_heads"], -1, BLOCK, c["dim"])
                scale = _scale_of(rows.abs().amax((-1, -2)))[..., None, None]
                y[i, :, :m] = (_e4m3((rows / scale).clamp(-448, 448)) * scale).flatten(1, 2)[:, :m]
        return [None, None, left, *out]
    k, v = c["beams"], c["vocab"]
    totals, states = [], [torch.empty_like(x) for x in s["states"]]
    for i in range(c["batch"]):
        x = torch.log_softmax(s["logits"][i * k : (i + 1) * k].double(), -1) + s["scores"][i].double()[:, None]
        for j in range(k):
            if int(s["ended"][i, j]):
                x[j] = -math.inf
                x[j, END] = s["scores"][i, j].double()
        best = torch.topk(x.reshape(-1), k)
        totals.append(best.values)
        at = torch.div(best.indices, v, rounding_mode="floor") + i * k  # (of equal logits of one beam: the same parent)
        for old, new in zip(s["states"], states):
            new[:, i * k : (i + 1) * k] = old[:, at]
    return [None, None, torch.stack(totals), None, *(x.double() if x.numel() < 1 << 28 else None for x in states)]
