"""The 8-bit block cache on the GPU: rows in and out, attention, eviction, against 64 bits (blocks_util)."""
import math

import pytest
import torch

from moondream_amd.block_cache import BlockCache
from moondream_amd.engine import no_collection

import blocks_util as U

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def random_rows(g, *shape, spread=2.0):
    """bf16 rows whose sizes differ: neighbouring blocks get different scales."""
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randn(*shape[:-1], 1, generator=g) * spread)
    return x.to(BF16)


def filled(g, slots, ctx, kv_heads, dim, spread=1.0, junk=None):
    """A cache of random rows (K, V in 64 bits beside it).  junk: a code that every row from there on holds, its blocks' scales too: (row, byte)."""
    c = BlockCache(slots, ctx, kv_heads, dim)
    k, v = (random_rows(g, slots, c.ctx, kv_heads, dim, spread=spread).cuda() for _ in range(2))
    c.append(k, v, ints([0] * slots))
    kk, vv = U.held(c.k.cpu(), c.k_exp.cpu()), U.held(c.v.cpu(), c.v_exp.cpu())
    if junk is not None:
        for s, row in enumerate(junk[0]):
            for t in (c.k, c.v):
                t[s, :, row:] = junk[1]
            for e in (c.k_exp, c.v_exp):
                e[s, :, (row + U.BLOCK - 1) // U.BLOCK :] = 255
    return c, kk, vv


# ------------------------------------------------------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 3, 32])
@pytest.mark.parametrize("tokens, row0, new", [(1, [0, 31, 32], None), (1, [95, 63, 5], None), (2, [31, 0, 94], None), (33, [0, 31, 17], None), (70, [1, 90, 26], None),
                                               (96, [0, 0, 0], [96, 1, 0]), (40, [10, -1, 200], [40, 40, 40]), (40, [95, 96, 60], [7, 5, -3])])
def test_appended_rows_are_the_definition_s(dim, heads, tokens, row0, new):
    g = torch.Generator().manual_seed(tokens * 131 + dim + heads)
    ctx, batch = 96, len(row0)
    c, k0, v0 = filled(g, batch, ctx, heads, dim)
    before = [t.clone() for t in (c.k, c.v, c.k_exp, c.v_exp)]
    qkv = random_rows(g, batch, tokens, 3 * heads + 1, dim, spread=3.0).cuda()  # keys and values are views of a projection's rows
    k, v = qkv[:, :, 1 : 1 + heads], qkv[:, :, 1 + 2 * heads :]
    c.append(k, v, ints(row0), new=None if new is None else ints(new))
    got_k, got_v = c.read(None, ctx)
    for x, vals, exps, got, after in ((k.cpu(), k0, before[2].cpu(), got_k.cpu(), c.k_exp.cpu()), (v.cpu(), v0, before[3].cpu(), got_v.cpu(), c.v_exp.cpu())):
        for b in range(batch):
            for h in range(heads):
                values, e = vals[b, h].clone(), (exps[b, h].int() - 127).tolist()
                U.append(values, e, x[b, :, h], row0[b], tokens if new is None else new[b])
                n = max(0, min(ctx, row0[b] + (tokens if new is None else new[b]))) if row0[b] >= 0 else 0
                assert (after[b, h].int() - 127).tolist() == e
                assert torch.equal(got[b, h, :n].double(), values[:n])
    for t, was, heads_ in ((c.k, before[0], heads), (c.v, before[1], heads)):  # rows behind the appended ones: the same bytes
        for b in range(batch):
            end = row0[b] + max(0, tokens if new is None else new[b])
            if 0 <= row0[b] and 0 <= end < ctx:
                assert torch.equal(t[b, :, end:], was[b, :, end:])


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_one_by_one_share_their_block_s_scale(dim):
    g = torch.Generator().manual_seed(5)
    c = BlockCache(1, 64, 2, dim)
    x = random_rows(g, 1, 40, 2, dim, spread=3.0).cuda()
    x[0, 20] *= 1000
    values, exps = torch.zeros(2, 64, dim, dtype=torch.float64), [[0, 0], [0, 0]]
    for t in range(40):
        c.append(x[:, t : t + 1], -x[:, t : t + 1], ints([t]))
        for h in range(2):
            U.append(values[h], exps[h], x[0, t : t + 1, h].cpu(), t, 1)
    k, v = c.read(None, 40)
    assert torch.equal(k[0].cpu().double(), values[:, :40]) and torch.equal(v, -k)


def test_zeros_infinities_and_nan_are_stored_as_numbers():
    c = BlockCache(1, 64, 1, 64)
    x = torch.zeros(1, 64, 1, 64)
    x[0, 0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 448.0])
    x[0, 33, 0, :3] = torch.tensor([2.0**-49, 2.0**-50, 2.0**-52])  # subnormal at the least scale: kept, a tie to even (0), 0
    x = x.to(BF16).cuda()
    c.append(x, x, ints([0]))
    k, _ = c.read(None, 64)
    assert k[0, 0, 0, :5].tolist() == [0.0, 448.0, -448.0, 448.0, 0.0]
    assert k[0, 0, 33, :3].tolist() == [2.0**-49, 0.0, 0.0]
    big = torch.full((1, 32, 1, 64), 3e38, dtype=BF16, device="cuda")
    c.append(big, big, ints([32]))
    assert float(c.read(None, 64)[0][0, 0, 40, 7]) == 448 * 2.0**U.HIGH


def test_reading_is_bounded_by_lengths_slots_and_the_cache():
    g = torch.Generator().manual_seed(6)
    c, k0, v0 = filled(g, 3, 64, 2, 64)
    k, v = c.read(ints([-3, 60, 5, 0]), 10, kv_len=ints([4, 64, 1000, -5]), slot=ints([2, 0, 1, 1]))
    for b, (slot, r0, n) in enumerate([(2, -3, 4), (0, 60, 64), (1, 5, 64), (1, 0, 0)]):
        for r in range(10):
            want = k0[slot, :, r0 + r] if 0 <= r0 + r < n else torch.zeros(2, 64, dtype=torch.float64)
            assert torch.equal(k[b, :, r].cpu().double(), want)
    k, v = c.read(ints([0, 0]), 5, slot=ints([-1, 3]))
    assert not bool(k.any()) and not bool(v.any())
    before = c.k.clone()
    x = torch.ones(2, 4, 2, 64, dtype=BF16, device="cuda")
    c.append(x, x, ints([0, 0]), slot=ints([3, -1]))
    assert torch.equal(before, c.k)


# ------------------------------------------------------------------------------------------------------------------------ attention
def attend(c, k, v, q, lens, *, q_pos0=None, q_rows=None, slot=None, prefix=0, scale=None, max_len=None, weights=False, decay=1.0, seed=0):
    """The kernel's outputs against 64 bits."""
    batch, tokens, heads, dim = q.shape
    g = torch.Generator().manual_seed(seed)
    w0 = torch.rand(c.slots, c.kv_heads, c.ctx, generator=g) if weights else None
    w = w0.cuda() if weights else None
    out = torch.full((batch, tokens, heads, dim), 7.0, dtype=BF16, device="cuda")
    opt = {n: ints(x) for n, x in (("q_pos0", q_pos0), ("q_rows", q_rows), ("slot", slot)) if x is not None}
    got = c.attention(q.cuda(), ints(lens), prefix_len=prefix, scale=scale, max_len=max_len, weights=w, decay=decay, out=out, **opt)
    assert got is out
    got = got.cpu().double()
    want_w = w0.double().clone() if weights else None
    for b in range(batch):
        s = slot[b] if slot is not None else b
        n = min(max(lens[b], 0), c.ctx if max_len is None else max_len, c.ctx) if 0 <= s < c.slots else 0
        rows = tokens if q_rows is None else min(max(q_rows[b], 0), tokens)
        pos0 = n - rows if q_pos0 is None else q_pos0[b]
        assert bool((got[b, rows:] == 7.0).all()), "a padding query's output changed"
        if rows == 0:
            o = torch.zeros(0, heads, dim, dtype=torch.float64)
            wt = torch.zeros(c.kv_heads, c.ctx, dtype=torch.float64)
            size, most, mass = o, 0.0, 0.0
        else:
            o, wt, size, most, mass = U.attention(q[b, :rows], k[s % c.slots], v[s % c.slots], n, pos0, prefix, scale if scale is not None else dim**-0.5)
        tol = U.attention_tolerance(o, size, most, mass, dim, n, float(v[s % c.slots, :, :n].abs().max()) if n else 0.0)
        assert bool((torch.isfinite(got[b, :rows])).all())
        worst = ((got[b, :rows] - o).abs() - tol)
        assert bool((worst <= 0).all()), f"sequence {b}: off by {float((got[b, :rows] - o).abs().max())}, {float(worst.max())} too much"
        if weights and n:
            want = decay * w0[s, :, :n].double() + wt[:, :n]
            t = U.weights_tolerance(wt[:, :n], most, mass, dim, rows * heads // c.kv_heads) + decay * w0[s, :, :n].double() * 2.0**-24 + want * 2.0**-23
            assert bool(((w[s, :, :n].cpu().double() - want).abs() <= t).all()), f"weights of sequence {b}: {float((w[s, :, :n].cpu().double() - want).abs().max())}"
            want_w[s, :, :n] = w[s, :, :n].cpu().double()
    if weights:
        assert torch.equal(w.cpu().double(), want_w), "weights of rows behind the last, or of other slots, changed"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads, group", [(1, 1), (3, 1), (2, 4), (1, 16), (2, 17), (1, 71)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_few_queries(dim, kv_heads, group, tokens):
    g = torch.Generator().manual_seed(dim + 7 * group + tokens)
    lens = [0, 1, 31, 32, 33, 127, 200, 256]
    c, k, v = filled(g, len(lens), 256, kv_heads, dim, junk=(lens, 0x7F))
    q = torch.randn(len(lens), tokens, kv_heads * group, dim, generator=g).to(BF16)
    attend(c, k, v, q, lens, weights=group in (1, 4, 17), decay=0.5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads, group, tokens", [(2, 1, 33), (1, 3, 100), (1, 8, 65), (2, 1, 300)])
def test_prompts(dim, kv_heads, group, tokens):
    g = torch.Generator().manual_seed(dim + group + tokens)
    lens = [tokens, tokens + 1, 320, 350, 317]
    c, k, v = filled(g, len(lens), 352, kv_heads, dim, junk=(lens, 0xFF))
    q = torch.randn(len(lens), tokens, kv_heads * group, dim, generator=g).to(BF16)
    attend(c, k, v, q, lens, weights=True, decay=0.0)
    attend(c, k, v, q, lens, prefix=64, max_len=350)
    attend(c, k, v, q, [0, 1, 5, 31, 32], weights=True)  # more queries than rows: the first ones see nothing


@pytest.mark.parametrize("tokens", [1, 5, 48])
@pytest.mark.parametrize("prefix", [0, 40, 1000])
def test_positions_padding_and_absent_sequences(tokens, prefix):
    g = torch.Generator().manual_seed(tokens + prefix)
    c, k, v = filled(g, 4, 128, 2, 64)
    q = torch.randn(6, tokens, 4, 64, generator=g).to(BF16)
    lens, slot = [100, 128, 77, 60, 50, 500], [3, 1, 1, -1, 4, 0]  # a slot that two sequences read, absent ones, a length past the cache
    attend(c, k, v, q, lens, slot=slot, prefix=prefix)
    attend(c, k, v, q, lens, slot=slot, prefix=prefix, q_rows=[tokens, 1, 0, tokens, 1, -4])
    attend(c, k, v, q, lens, slot=slot, prefix=prefix, q_pos0=[0, 127, -3, 5, 5, 2000], max_len=90)
    attend(c, k, v, q[:4], [100, 128, 77, 60], slot=[2, 0, 1, 3], prefix=prefix, q_rows=[1, tokens, 0, tokens], weights=True)


@pytest.mark.parametrize("dim, kv_heads, group, tokens, ctx", [(64, 8, 1, 200, 2300), (128, 8, 2, 150, 2100), (64, 3, 5, 90, 2400), (64, 1, 130, 3, 2100)])
def test_ragged_batches_of_long_prompts(dim, kv_heads, group, tokens, ctx):
    """Workgroups in the order of their reach: sequences of every length, padded, absent and empty ones among them, prefixes; more heads in a group than columns in a workgroup."""
    g = torch.Generator().manual_seed(ctx + dim)
    c, k, v = filled(g, 6, ctx, kv_heads, dim)
    q = torch.randn(7, tokens, kv_heads * group, dim, generator=g).to(BF16)
    lens, slot = [ctx, 300, 0, tokens, ctx - 1, 1111, 700], [0, 1, 2, 5, 4, 3, 6]
    rows = [tokens, 1, tokens, tokens // 2, tokens - 1, 0, tokens]
    attend(c, k, v, q, lens, slot=slot, q_rows=rows, weights=True, decay=0.25)
    attend(c, k, v, q, lens, slot=slot, q_rows=rows, prefix=600, q_pos0=[50, 0, 5, ctx, -10, 1000, 0])


def test_more_sequences_than_a_wave_has_lanes():
    g = torch.Generator().manual_seed(70)
    c, k, v = filled(g, 3, 2080, 1, 64)
    q = torch.randn(70, 40, 1, 64, generator=g).to(BF16)
    attend(c, k, v, q, [2080 - 29 * i for i in range(70)], slot=[i % 3 for i in range(70)], q_rows=[40 - i % 5 for i in range(70)])


@pytest.mark.parametrize("dim, group", [(64, 1), (64, 17), (128, 1), (128, 20)])
@pytest.mark.parametrize("batch, kv_heads, length", [(1, 2, 700), (9, 16, 1200), (30, 10, 520)])
def test_few_queries_over_short_caches_in_one_launch_and_in_two(dim, group, batch, kv_heads, length):
    g = torch.Generator().manual_seed(batch + dim + group)
    slots = min(batch, 4)
    c, k, v = filled(g, slots, length, kv_heads, dim)
    q = torch.randn(batch, 1, kv_heads * group, dim, generator=g).to(BF16)
    slot, lens = [i % slots for i in range(batch)], [max(0, length - 37 * i) for i in range(batch)]
    attend(c, k, v, q, lens, slot=slot)
    if batch <= slots:
        attend(c, k, v, q, lens, slot=slot, weights=True, decay=0.0)


def test_negative_and_no_scale():
    g = torch.Generator().manual_seed(2)
    c, k, v = filled(g, 2, 100, 2, 64)
    for tokens in (1, 40):
        q = torch.randn(2, tokens, 2, 64, generator=g).to(BF16)
        attend(c, k, v, q, [100, 61], scale=-0.2, weights=True)
        attend(c, k, v, q, [100, 61], scale=0.0, weights=True)


def test_strided_queries_and_outputs():
    g = torch.Generator().manual_seed(1)
    c, k, v = filled(g, 2, 64, 2, 64)
    rows = torch.randn(3, 2, 12, 64, generator=g).to(BF16).cuda()  # [tokens, batch, heads, dim]
    q = rows.transpose(0, 1)[:, :, 2:10:2]
    full = torch.zeros(2, 4, 3, 64, dtype=BF16, device="cuda")
    out = full.transpose(1, 2)
    assert c.attention(q, ints([50, 64]), out=out) is out
    want = c.attention(q.contiguous(), ints([50, 64]))
    assert torch.equal(out.contiguous(), want)
    again = q.contiguous()
    assert c.attention(again, ints([50, 64]), out=again) is again and torch.equal(again, want)  # in the queries' place


@pytest.mark.parametrize("dim, kv_heads, group, tokens, length", [(64, 2, 1, 1, 5003), (64, 1, 8, 1, 9001), (128, 1, 4, 1, 7777), (128, 2, 2, 40, 4001), (64, 1, 1, 500, 3011)])
def test_long_caches(dim, kv_heads, group, tokens, length):
    """Keys over many workgroups."""
    g = torch.Generator().manual_seed(length)
    c, k, v = filled(g, 2, length, kv_heads, dim)
    q = torch.randn(2, tokens, kv_heads * group, dim, generator=g).to(BF16)
    attend(c, k, v, q, [length, length // 3], weights=True, decay=0.9)


@pytest.mark.parametrize("tokens", [1, 40])
def test_blocks_of_very_different_scales(tokens):
    """Values from 2^-30 to 2^30 in turn, and the weight on the smallest ones: fp16 holds a weight times its block's scale over the largest such product, so the small
    blocks' values come out whole where the large ones get no weight."""
    g = torch.Generator().manual_seed(3)
    c = BlockCache(1, 256, 1, 64)
    k, v = torch.randn(1, 256, 1, 64, generator=g), torch.randn(1, 256, 1, 64, generator=g)
    for i in range(8):
        v[:, 32 * i : 32 * i + 32] *= 2.0 ** ((-30, 30)[i % 2])
        k[:, 32 * i : 32 * i + 32, :, 0] = (60.0, -60.0)[i % 2]
    c.append(k.to(BF16).cuda(), v.to(BF16).cuda(), ints([0]))
    kk, vv = U.held(c.k.cpu(), c.k_exp.cpu()), U.held(c.v.cpu(), c.v_exp.cpu())
    q = torch.randn(1, tokens, 1, 64, generator=g)
    q[..., 0] = 8.0
    q = q.to(BF16)
    got = c.attention(q.cuda(), ints([256]), scale=1.0).cpu().double()
    o, _, size, most, mass = U.attention(q[0], kk[0], vv[0], 256, 256 - tokens, 0, 1.0)
    assert 0 < float(o.abs().max()) < 2.0**-26
    tol = U.attention_tolerance(o, size, most, mass, 64, 256, float(vv[0, :, :32].abs().max()))
    assert bool(((got[0] - o).abs() <= tol).all())


def test_extreme_scores_stay_finite_and_nan_queries_stay_alone():
    g = torch.Generator().manual_seed(4)
    c, k, v = filled(g, 2, 96, 1, 64)
    q = torch.randn(2, 4, 1, 64, generator=g).to(BF16)
    attend(c, k, v, q, [96, 70], scale=-300.0)
    q[0, 1, 0, 5] = math.nan
    q[1, 2, 0, 7] = math.inf
    got = c.attention(q.cuda(), ints([96, 70]))
    clean = c.attention(torch.nan_to_num(q, 0, 0, 0).cuda(), ints([96, 70]))
    for b, bad in ((0, 1), (1, 2)):
        for t in range(4):
            if t == bad:
                assert bool(torch.isnan(got[b, t]).all())
            else:
                assert torch.equal(got[b, t], clean[b, t])


def test_offsets_past_32_bits():
    """The last slot of a cache of over 4 GiB of keys."""
    slots, heads, ctx = 70, 32, 32768
    c = BlockCache(slots, ctx, heads, 64)
    assert c.k.numel() > 1 << 32
    g = torch.Generator().manual_seed(8)
    x = random_rows(g, 1, 40, heads, 64).cuda()
    last = ints([slots - 1])
    c.append(x, x.flip(1), ints([ctx - 40]), slot=last)
    k, v = c.read(ints([ctx - 40]), 40, slot=last)
    first = c.read(ints([ctx - 40]), 40, slot=ints([0]))
    assert not bool(first[0].any())
    q = torch.randn(1, 1, heads, 64, generator=g).to(BF16)
    got = c.attention(q.cuda(), ints([ctx]), slot=last).cpu().double()
    # every other row is zero: weight exp(0), value zero
    t = torch.einsum("hd,hrd->hr", q[0, 0].double(), k[0].cpu().double()) / 8
    e = torch.exp(t)
    o = (e[..., None] * v[0].cpu().double()).sum(1) / (e.sum(1) + ctx - 40)[:, None]
    size = (e[..., None] * v[0].cpu().double().abs()).sum(1) / (e.sum(1) + ctx - 40)[:, None]
    mass = float(torch.einsum("hd,hrd->hr", q[0, 0].double().abs(), k[0].cpu().double().abs()).max() / 8)
    # the zero rows' products are exact, so subnormal fp16 weights (2^-25 of the largest product each) count for the 40 rows alone, at their largest value
    tol = U.attention_tolerance(o, size, float(t.abs().max()), mass, 64, 40, float(v.abs().max())) + size * ctx * 2.0**-23
    assert bool(((got[0, 0] - o).abs() <= tol).all())
    w = torch.zeros(slots, heads, ctx, device="cuda")
    w[slots - 1, :, ctx - 40 :] = 1.0
    kept, n = c.evict(w, ints([ctx]), 40, slot=last)
    assert torch.equal(kept[0, 0].cpu(), torch.arange(ctx - 40, ctx, dtype=I32)) and n.tolist() == [40]
    k2, v2 = c.read(ints([0]), 40, slot=last)
    for was, now in ((k[0].cpu().double(), k2[0]), (v[0].cpu().double(), v2[0])):  # (rows of two blocks share one now: as the definition rounds them)
        for h in range(heads):
            for b0 in (0, 32):
                e = U.exponent(U.finite_top(was[h, b0 : b0 + 32]))
                assert torch.equal(now[h, b0 : b0 + 32].cpu().double(), U.e4m3(was[h, b0 : b0 + 32] * 2.0**-e) * 2.0**e)


def test_one_head_past_32_bits():
    """A single head whose keys take over 4 GiB; the last rows outweigh the 67 million zeros before them."""
    ctx, n = (1 << 26) + 96, 70
    c = BlockCache(1, ctx, 1, 64)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, n, 1, 64, generator=g)
    x[..., 0] = 16.0
    x = x.to(BF16).cuda()
    c.append(x, x.flip(1), ints([ctx - n]))
    k, v = (r[0].cpu().double() for r in c.read(ints([ctx - n]), n))
    w = torch.zeros(1, 1, ctx, device="cuda")
    for tokens in (1, 40):
        q = torch.randn(1, tokens, 1, 64, generator=g)
        q[..., 0] = 24.0
        q = q.to(BF16)
        got = c.attention(q.cuda(), ints([ctx]), weights=w, decay=0.0).cpu().double()
        t = q[0, :, 0].double() @ k[0].T / 8
        seen = torch.arange(n)[None] <= torch.arange(n - tokens, n)[:, None]
        e = torch.where(seen, torch.exp(t), 0.0)
        zeros = ctx - n
        p = e / (e.sum(1, keepdim=True) + zeros)
        o, size = p @ v[0], p @ v[0].abs()
        mass = float((q[0, :, 0].double().abs() @ k[0].abs().T / 8).max())
        tol = U.attention_tolerance(o, size, float(t.abs().max()), mass, 64, n, float(v.abs().max())) + size * 2.0**-20
        assert bool(((got[0, :, 0] - o).abs() <= tol).all())
        near = (w[0, 0, ctx - n :].cpu().double() - p.sum(0)).abs()
        assert bool((near <= U.weights_tolerance(p.sum(0), float(t.abs().max()), mass, 64, tokens) + p.sum(0) * 2.0**-20).all())
    into, into_w = BlockCache(1, 96, 1, 64), torch.zeros(1, 1, 96, device="cuda")
    kept, length = c.evict(w, ints([ctx]), 64, recent=1, into=into, into_weights=into_w)
    best = torch.sort(w[0, 0, ctx - n : ctx - 1].cpu(), descending=True, stable=True).indices[:63]
    rows = torch.cat([best.sort().values, torch.tensor([n - 1])]) + ctx - n
    assert torch.equal(kept[0, 0].cpu().long(), rows) and length.tolist() == [64] and torch.equal(into_w[0, 0, :64].cpu(), w[0, 0].cpu()[rows])


# ------------------------------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("ctx, lens, keep, first, recent", [(96, [96, 50, 33, 1, 0], 33, 0, 0), (160, [160, 159, 100, 64, 65], 64, 4, 60), (160, [160, 31, 32, 33, -2], 32, 1, 7),
                                                            (1500, [1500, 1499, 700, 513, 9999], 513, 4, 100), (2240, [2240, 1800, 40, 2000, 1088], 1087, 0, 1),
                                                            (64, [64, 64, 1, 2, 3], 1, 0, 1), (64, [64, 63, 33, 32, 0], 64, 10, 10)])
def test_what_stays_and_how(dim, in_place, ctx, lens, keep, first, recent):
    g = torch.Generator().manual_seed(ctx + keep + dim)
    heads, slots = 3, 6
    c, k, v = filled(g, slots, ctx, heads, dim, spread=3.0)
    w = torch.randint(0, 8, (slots, heads, c.ctx), generator=g).float() * 0.25  # many ties
    w[0, 0, :5] = math.nan
    w[1, 1] = 0.0
    w[2, 2, 3] = math.inf
    w[0, 2] = torch.randn(c.ctx, generator=g)
    slot = [5, 0, 3, 2, 1]
    gw = w.cuda()
    into = None if in_place else BlockCache(slots, keep + 40, heads, dim)
    into_w = None if in_place else torch.full((slots, heads, into.ctx), 9.0, device="cuda")
    to = c if in_place else into
    before = [t.clone() for t in (to.k, to.v)]
    kept, n = c.evict(gw, ints(lens), keep, first=first, recent=recent, slot=ints(slot), into=into, into_weights=into_w)
    got_w = (gw if in_place else into_w).cpu()
    rk, rv = (x.cpu().double() for x in to.read(None, to.ctx))
    for b, s in enumerate(slot):
        length = min(max(lens[b], 0), c.ctx)
        m = min(length, keep)
        assert int(n[b]) == m
        for h in range(heads):
            rows = U.kept_rows(w[s, h].tolist(), length, keep, first, recent)
            assert kept[b, h].tolist() == rows + [-1] * (keep - m)
            assert torch.equal(torch.nan_to_num(got_w[s, h, :m], nan=-5.0), torch.nan_to_num(w[s, h][rows], nan=-5.0))
            if not in_place:
                assert bool((got_w[s, h, m:] == 9.0).all())
            for old, new, exps in ((k, rk, to.k_exp), (v, rv, to.v_exp)):
                for b0 in range(0, m, U.BLOCK):
                    x = old[s, h][rows[b0 : b0 + U.BLOCK]]
                    e = U.exponent(U.finite_top(x))
                    assert int(exps[s, h, b0 // U.BLOCK]) - 127 == e
                    assert torch.equal(new[s, h, b0 : b0 + len(x)], U.e4m3(x * 2.0**-e) * 2.0**e)
        for t, was in zip((to.k, to.v), before):
            if not in_place:
                assert torch.equal(t[s, :, m:], was[s, :, m:])
    assert torch.equal(to.k[4], before[0][4])  # a slot that no sequence has


@pytest.mark.parametrize("ctx, keep", [(4096, 1000), (4128, 4000), (40000, 5000), (70016, 33000)])
def test_rows_that_stay_of_long_caches(ctx, keep):
    """Weights held in registers, in one portion and in several; many equal ones at the border."""
    g = torch.Generator().manual_seed(keep)
    c = BlockCache(2, ctx, 2, 64)
    c.k.random_(0, 120)
    c.v.random_(0, 120)
    w = torch.exp(2 * torch.randn(2, 2, ctx, generator=g))
    w[0, 1] = torch.randint(0, 50, (ctx,), generator=g).float()
    w[1, 0, ::3] = 0.75
    lens = [ctx, ctx - 1234]
    buf = torch.zeros(2 * 2 * ctx + 1, device="cuda")  # an address that is no multiple of 16
    gw = buf[1:].view(2, 2, ctx)
    gw.copy_(w)
    kept, n = c.evict(gw, ints(lens), keep, first=3, recent=50, into=BlockCache(2, keep, 2, 64))
    for b in range(2):
        for h in range(2):
            x = w[b, h, : lens[b]].clone()
            x[:3] = x[lens[b] - 50 :] = math.inf
            best = torch.sort(x, descending=True, stable=True).indices[:keep].sort().values
            assert torch.equal(kept[b, h, : len(best)].cpu().long(), best) and bool((kept[b, h, len(best) :] == -1).all())


def test_outputs_that_share_memory_are_refused():
    c, _, _ = filled(torch.Generator().manual_seed(14), 2, 64, 2, 64)
    q = torch.zeros(2, 3, 4, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        c.attention(q, ints([5, 6]), out=torch.zeros(2, 1, 4, 64, dtype=BF16, device="cuda").expand(2, 3, 4, 64))


def test_another_longest_in_every_step():
    c, _, _ = filled(torch.Generator().manual_seed(15), 1, 2048, 1, 64)
    q, n = torch.randn(1, 1, 1, 64, device="cuda").to(BF16), ints([9])
    first = c.attention(q, n)
    for longest in range(900, 2048):
        out = c.attention(q, n, max_len=longest)
    assert torch.equal(out, first) and len(c._workspaces) <= 1024


@pytest.mark.parametrize("ctx", [96, 8192])
def test_zeros_of_both_signs_are_equal_weights(ctx):
    c = BlockCache(1, ctx, 1, 64)
    w = torch.zeros(1, 1, ctx)
    w[0, 0, 1::2] = 0.0
    w[0, 0, ::2] = -0.0
    w[0, 0, 40] = -1e-30
    w[0, 0, 50] = 1e-45
    kept, n = c.evict(w.cuda(), ints([ctx]), 45)
    assert kept[0, 0].tolist() == [j for j in range(45) if j != 40] + [50] and n.tolist() == [45]


def test_eviction_in_place_is_the_same_as_into_another_cache():
    g = torch.Generator().manual_seed(11)
    c, k, v = filled(g, 2, 6000, 2, 64, spread=2.0)
    w = torch.rand(2, 2, c.ctx, generator=g).cuda()
    into, into_w = BlockCache(2, 4500, 2, 64), torch.zeros(2, 2, 4512, device="cuda")
    lens = ints([6000, 5555])
    kept, n = c.evict(w, lens, 4500, recent=100, into=into, into_weights=into_w)
    kept2, n2 = c.evict(w, lens, 4500, recent=100)
    assert torch.equal(kept, kept2) and torch.equal(n, n2) and torch.equal(w[:, :, :4500], into_w[:, :, :4500])
    for a, b in zip(c.read(None, 4500), into.read(None, 4500)):
        assert torch.equal(a, b)


def test_eviction_of_absent_sequences_touches_nothing():
    g = torch.Generator().manual_seed(12)
    c, _, _ = filled(g, 2, 64, 1, 64)
    w = torch.rand(2, 1, 64, device="cuda")
    before = c.k.clone(), w.clone()
    kept, n = c.evict(w, ints([64, 64]), 8, slot=ints([1, 5]), into=BlockCache(1, 64, 1, 64))  # a slot that the other cache does not have
    assert n.tolist() == [0, 0] and bool((kept == -1).all())
    kept, n = c.evict(w, ints([64, 64]), 8, slot=ints([-1, 2]))
    assert n.tolist() == [0, 0] and bool((kept == -1).all()) and torch.equal(before[0], c.k) and torch.equal(before[1], w)


def test_python_refuses_what_does_not_fit():
    g = torch.Generator().manual_seed(13)
    c, _, _ = filled(g, 2, 64, 2, 64)
    x, q, n = torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda"), torch.zeros(2, 3, 4, 64, dtype=BF16, device="cuda"), ints([5, 6])
    w = torch.zeros(2, 2, 64, device="cuda")
    calls = [lambda: c.append(x.float(), x, n), lambda: c.append(x, x[:, :2], n), lambda: c.append(x[:, :, :1], x, n), lambda: c.append(x, x, n.long()), lambda: c.append(x, x, n.cpu()),
             lambda: c.append(x, x, n[:1]), lambda: c.append(x.cpu(), x, n), lambda: c.append(x.transpose(2, 3).contiguous().transpose(2, 3), x, n), lambda: c.append(x, x, n, new=n[:1]),
             lambda: c.append(torch.cat([x, x]), torch.cat([x, x]), ints([0] * 4)), lambda: c.append(x[:, :, :, :32], x, n), lambda: c.read(n, -1), lambda: c.read(ints([0] * 3), 4),
             lambda: c.attention(q[:, :, :3], n), lambda: c.attention(q.float(), n), lambda: c.attention(q, n, max_len=0), lambda: c.attention(q, n, prefix_len=-1),
             lambda: c.attention(q, n, weights=w[:, :1]), lambda: c.attention(q, n, weights=w.double()), lambda: c.attention(q, n, out=q[:, :2]), lambda: c.attention(q, n, slot=n.long()),
             lambda: c.attention(q, n, weights=w.transpose(1, 2)), lambda: c.evict(w, n, 0), lambda: c.evict(w, n, 65), lambda: c.evict(w, n, 8, first=5, recent=4),
             lambda: c.evict(w, n, 8, into=BlockCache(2, 64, 1, 64)), lambda: c.evict(w, n, 8, into_weights=w), lambda: c.evict(w, n, 8, into=BlockCache(1, 64, 2, 64)),
             lambda: c.evict(w, n, 64, into=BlockCache(2, 32, 2, 64)), lambda: c.evict(w[0], n, 8)]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    from moondream_amd._lib import MoondreamHipError

    with pytest.raises(MoondreamHipError):
        c.attention(q, n, scale=math.nan)
    with pytest.raises(MoondreamHipError):
        c.evict(w, n, 8, into=BlockCache.of(c.k, c.v, c.k_exp.clone(), c.v_exp))
    assert c.attention(q[:, :0], n).shape == (2, 0, 4, 64) and c.read(n, 0)[0].shape == (2, 2, 0, 64)
    c.append(x[:, :0], x[:, :0], n)


def test_another_layers_slab_and_a_stream_of_its_own():
    """Slots that lie apart (a layer's part of a slab of all layers), calls on another stream than the current one's."""
    g = torch.Generator().manual_seed(14)
    whole = [torch.zeros(3, 2, 2, 64, 64, dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.full((3, 2, 2, 2), 127, dtype=torch.uint8, device="cuda") for _ in range(2)]
    layers = [BlockCache.of(*(t[:, i] for t in whole)) for i in range(2)]
    x, y = random_rows(g, 3, 50, 2, 64).cuda(), random_rows(g, 3, 50, 2, 64).cuda()
    q = torch.randn(3, 1, 2, 64, generator=g).to(BF16).cuda()
    n = ints([50, 50, 50])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layers[1].append(x, y, ints([0, 0, 0]))
        got = layers[1].attention(q, n)
    torch.cuda.current_stream().wait_stream(side)
    alone = BlockCache(3, 64, 2, 64)
    alone.append(x, y, ints([0, 0, 0]))
    assert torch.equal(got, alone.attention(q, n))
    assert not bool(whole[0][:, 0].any())


def test_results_do_not_hang_on_the_batch_or_the_run():
    g = torch.Generator().manual_seed(15)
    c, _, _ = filled(g, 8, 3000, 2, 64)
    q = torch.randn(8, 1, 8, 64, generator=g).to(BF16).cuda()
    lens = [3000, 2999, 100, 1, 2048, 31, 500, 2500]
    w = torch.zeros(8, 2, c.ctx, device="cuda")
    a = c.attention(q, ints(lens), weights=w, decay=0.0)
    for _ in range(3):
        w2 = torch.zeros_like(w)
        assert torch.equal(a, c.attention(q, ints(lens), weights=w2, decay=0.0)) and torch.equal(w, w2)


def test_a_captured_step_replays_as_it_runs():
    """append, attention with weights and eviction in one graph, replayed several times between eager work; two graphs in turn on one cache."""
    g = torch.Generator().manual_seed(16)
    heads, dim, ctx = 2, 64, 256
    caches = [BlockCache(2, ctx, heads, dim) for _ in range(2)]
    start = random_rows(g, 2, 100, heads, dim).cuda()
    for c in caches:
        c.append(start, start.flip(1), ints([0, 0]))
    state = [dict(len=ints([100, 90]), w=torch.zeros(2, heads, ctx, device="cuda")) for _ in caches]
    k, v, q = (torch.zeros(2, 1, n, dim, dtype=BF16, device="cuda") for n in (heads, heads, 4))
    outs = {}

    def step(i):
        c, s = caches[i], state[i]
        c.append(k, v, s["len"])
        s["len"] += 1
        o = c.attention(q, s["len"], weights=s["w"], max_len=ctx)
        kept, n = c.evict(s["w"], s["len"], 96, first=2, recent=20)
        s["len"].copy_(n)
        return o, kept

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    saved = [(c.k.clone(), c.v.clone(), c.k_exp.clone(), c.v_exp.clone(), s["len"].clone(), s["w"].clone()) for c, s in zip(caches, state)]
    with torch.cuda.stream(side):
        step(0)  # a first run outside of a capture
        for t, was in zip((caches[0].k, caches[0].v, caches[0].k_exp, caches[0].v_exp, state[0]["len"], state[0]["w"]), saved[0]):
            t.copy_(was)
    torch.cuda.current_stream().wait_stream(side)
    with no_collection():
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs[len(graphs)] = step(0)
            graphs.append(graph)
    torch.cuda.synchronize()
    for t, was in zip((caches[0].k, caches[0].v, caches[0].k_exp, caches[0].v_exp, state[0]["len"], state[0]["w"]), saved[0]):
        t.copy_(was)
    for i in range(6):
        for t, n in ((k, heads), (v, heads), (q, 4)):
            t.copy_(random_rows(g, 2, 1, n, dim))
        o, kept = step(1)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        go, gkept = outs[i % 2]
        assert torch.equal(o, go) and torch.equal(kept, gkept), f"replay {i}"
        assert torch.equal(state[0]["w"], state[1]["w"]) and torch.equal(state[0]["len"], state[1]["len"]) and torch.equal(caches[0].k, caches[1].k)
