"""Beam search on the GPU: the choice against 64 bits, states behind their parents, and a whole search over the 8-bit cache."""
import math

import pytest
import torch

from moondream_amd.beams import reorder_states, select_beams
from moondream_amd.block_cache import BlockCache
from moondream_amd.engine import no_collection

import blocks_util as U

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16


def check(logits, scores, ended=None, end_id=-1, suppress_id=-1, rank_weight=None):
    batch, beams = scores.shape
    got = select_beams(logits.cuda(), scores.cuda(), ended=None if ended is None else ended.cuda(), end_id=end_id, suppress_id=suppress_id,
                       rank_weight=None if rank_weight is None else rank_weight.cuda())
    for b in range(batch):
        want = U.beams(logits[b * beams : (b + 1) * beams], scores[b], None if ended is None else ended[b], end_id, suppress_id, None if rank_weight is None else rank_weight[b])
        assert got.tokens[b].tolist() == [w[0] for w in want]
        assert got.parents[b].tolist() == [w[1] for w in want]
        assert got.ended[b].tolist() == [w[3] for w in want]
        for x, w in zip(got.scores[b].tolist(), want):
            # totals are rounded to fp32 once; the sum of exponentials: fp32 exponentials of arguments of a few units, 2^-21 at most
            assert x == w[2] or abs(x - w[2]) <= abs(w[2]) * 2.0**-24 + 2.0**-21, (x, w[2])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("vocab", [2, 7, 255, 8191, 8192, 8193, 51200, 70001])
@pytest.mark.parametrize("batch, beams", [(1, 2), (3, 4), (2, 5), (2, 16)])
def test_choices(dtype, vocab, batch, beams):
    g = torch.Generator().manual_seed(vocab + beams)
    logits = (torch.randn(batch * beams, vocab, generator=g) * 3).to(dtype)
    scores = -torch.rand(batch, beams, generator=g) * 5
    ended = (torch.rand(batch, beams, generator=g) < 0.3).to(I32)
    check(logits, scores)
    check(logits, scores, ended=ended, end_id=vocab - 1, suppress_id=1)
    check(logits, scores, ended=ended, end_id=0, rank_weight=torch.rand(batch, beams, generator=g) + 0.5)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_a_search_begins_with_one_beam(dtype):
    g = torch.Generator().manual_seed(0)
    row = torch.randn(1, 9000, generator=g).to(dtype)
    scores = torch.full((2, 4), -math.inf)
    scores[:, 0] = 0
    check(row.expand(8, -1).contiguous(), scores)


def test_ties_go_to_the_lower_beam_and_token():
    logits = torch.zeros(6, 20000)
    logits[:, [19999, 8192, 5, 8191]] = 2.0
    got = select_beams(logits.cuda(), torch.zeros(2, 3).cuda())
    assert got.tokens.tolist() == [[5, 8191, 8192]] * 2 and got.parents.tolist() == [[0, 0, 0]] * 2
    logits[:, 5] = -0.0
    logits[:, [19999, 8192, 8191]] = 0.0  # all equal now, negative zero among them
    assert select_beams(logits.cuda(), torch.zeros(2, 3).cuda()).tokens.tolist() == [[0, 1, 2]] * 2


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_many_pieces_and_many_rows(dtype):
    g = torch.Generator().manual_seed(7)
    check((torch.randn(4, 300007, generator=g) * 2).to(dtype), -torch.rand(2, 2, generator=g))  # more pieces than a wave has lanes
    check((torch.randn(16, 300007, generator=g) * 2).to(dtype), -torch.rand(1, 16, generator=g))  # ... and than lists have room
    logits = (torch.randn(256, 8200, generator=g) * 2).to(dtype)
    logits[3], logits[17], logits[40:56] = 1.0, logits[17].round(), logits[40:56].clamp(max=2.0)  # more equal logits than are put in order together
    check(logits, -torch.rand(16, 16, generator=g), suppress_id=8199)


def test_what_is_no_number():
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(8, 300, generator=g)
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 10:] = -math.inf
    logits[3, 7] = math.inf
    logits[4, ::2] = math.nan
    logits[5, 1:] = -math.inf
    scores = torch.tensor([[-1.0, -2.0, -3.0, -30.0], [-1.0, math.nan, -math.inf, -2.0]])
    check(logits, scores)
    check(logits, scores, ended=torch.tensor([[0, 0, 1, 0], [0, 1, 1, 0]], dtype=I32), end_id=3)
    weight = torch.tensor([[1.0, 1.0, math.nan, 0.5], [math.inf, 1.0, 1.0, 1.0]])  # beams whose weighted totals are no numbers have no continuations
    got = select_beams(logits.cuda(), scores.cuda(), rank_weight=weight.cuda(), end_id=3)
    alive = scores.clone()
    alive[0, 2] = alive[1, 0] = -math.inf
    for a, b in zip(got, select_beams(logits.cuda(), alive.cuda(), rank_weight=torch.nan_to_num(weight, 1.0, 1.0).cuda(), end_id=3)):
        assert torch.equal(a, b)
    dead = torch.full((1, 3), -math.inf)
    got = select_beams(logits[:3].cuda(), dead.cuda(), end_id=9)
    assert got.tokens.tolist() == [[9] * 3] and got.parents.tolist() == [[0, 1, 2]] and got.ended.tolist() == [[1] * 3] and bool((got.scores == -math.inf).all())
    one = torch.full((2, 50), -math.inf)
    one[0, 4] = 3.0
    got = select_beams(one.cuda(), torch.zeros(1, 2).cuda())
    assert got.tokens.tolist() == [[4, -1]] and got.parents.tolist() == [[0, 1]] and got.scores.tolist() == [[0.0, -math.inf]]


@pytest.mark.parametrize("dtype, offset, extra", [(BF16, 0, 8), (BF16, 1, 0), (BF16, 3, 5), (torch.float32, 1, 3), (torch.float32, 2, 4)])
def test_rows_of_any_alignment(dtype, offset, extra):
    g = torch.Generator().manual_seed(offset)
    buf = torch.randn(8, 10001 + offset + extra, generator=g).to(dtype)
    logits, scores = buf[:, offset : offset + 10001], -torch.rand(2, 4, generator=g)
    got = select_beams(buf.cuda()[:, offset : offset + 10001], scores.cuda())
    want = select_beams(logits.contiguous().cuda(), scores.cuda())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    check(logits.contiguous(), scores)


@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 16])
@pytest.mark.parametrize("in_place", [False, True])
def test_states_follow_their_parents(beams, in_place):
    g = torch.Generator().manual_seed(beams)
    batch = 3
    n = batch * beams
    parents = torch.randint(0, beams, (batch, beams), generator=g)
    parents[0] = torch.arange(beams).flip(0)  # swaps
    parents[1] = torch.arange(beams)  # nothing moves
    slots = (parents + torch.arange(batch)[:, None] * beams).reshape(-1)
    shapes = [((n, 5, 16), BF16), ((n + 2, 3), torch.float32), ((n,), torch.uint8), ((n, 7, 9), torch.uint8), ((n, 4, 64, 32), torch.float32)]
    states = [torch.randint(0, 200, s, generator=g).to(t).cuda() for s, t in shapes] * 9  # more pieces than one launch takes
    states = [s.clone() for s in states]
    slab = torch.randn(3, n, 2, 40, 64, generator=g).to(BF16).cuda()
    wants = [torch.cat([s[slots], s[n:]]) for s in states]
    want_slab = slab.clone()
    want_slab[:, :, :, 7:23] = slab[:, slots][:, :, :, 7:23]
    p = parents.to(I32).cuda()
    if in_place:
        reorder_states(states, p)
        got = states
        reorder_states([slab[:, :, :, 7:23]], p, slot_dim=1)
        assert torch.equal(slab, want_slab)
    else:
        got = [torch.zeros_like(s) for s in states]
        for o, s in zip(got, states):
            o[n:] = s[n:]
        reorder_states(states, p, into=got)
        other = slab.clone()
        reorder_states([slab[:, :, :, 7:23]], p, into=[other[:, :, :, 7:23]], slot_dim=1)
        assert torch.equal(other, want_slab)
    for a, b in zip(got, wants):
        assert torch.equal(a, b)


def test_parents_out_of_range_move_nothing():
    x = torch.arange(8.0, device="cuda").view(4, 2)
    want = x.clone()
    reorder_states([x], torch.tensor([[-1, 2], [1 << 30, -(1 << 31)]], dtype=I32, device="cuda"))
    assert torch.equal(x, want)


def test_states_past_32_bits():
    x = torch.zeros(4, (1 << 30) + 64, dtype=torch.uint8, device="cuda")
    for i in range(4):
        x[i, -64:] = i + 1
        x[i, :64] = 10 + i
    reorder_states([x], torch.tensor([[3, 0, 2, 1]], dtype=I32, device="cuda"))
    assert x[:, -1].tolist() == [4, 1, 3, 2] and x[:, 0].tolist() == [13, 10, 12, 11] and not bool(x[:, 64:-64:4097].any())


def test_captured_calls_replay_and_streams_do_not_disturb_one_another():
    """A portion of prompts with weights, a choice and a reordering in two graphs over the same inputs, replayed in turn, between eager runs and beside work on another stream."""
    g = torch.Generator().manual_seed(21)
    cache = BlockCache(4, 640, 2, 64)
    rows = torch.randn(4, 640, 2, 64, generator=g).to(BF16).cuda()
    cache.append(rows, rows.flip(1), torch.zeros(4, dtype=I32, device="cuda"))
    q, length = torch.randn(4, 300, 4, 64, generator=g).to(BF16).cuda(), torch.tensor([640, 500, 301, 640], dtype=I32, device="cuda")
    logits, scores = torch.randn(8, 9000, generator=g).cuda(), -torch.rand(2, 4, generator=g).cuda()
    state = torch.randn(3, 8, 2, 40, generator=g).cuda()

    def work(w, into):
        o = cache.attention(q, length, weights=w, decay=0.0)
        choice = select_beams(logits, scores, end_id=5)
        reorder_states([state], choice.parents, into=[into], slot_dim=1)
        return (o, *choice)

    buffers = [(torch.zeros(4, 2, 640, device="cuda"), torch.zeros_like(state)) for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(*buffers[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    with no_collection():
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(work(*buffers[i]))
            graphs.append(graph)
    for turn in range(4):
        for t in (q, logits, state):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            beside = work(*buffers[3])
        graphs[turn % 2].replay()
        eager = work(*buffers[2])
        torch.cuda.synchronize()
        for a, b, c in zip((*outs[turn % 2], *buffers[turn % 2]), (*eager, *buffers[2]), (*beside, *buffers[3])):
            assert torch.equal(a, b) and torch.equal(c, b), f"turn {turn}"


@pytest.mark.parametrize("beams, dim, group", [(4, 64, 1), (3, 128, 4)])
def test_a_search_over_the_block_cache(beams, dim, group):
    """A layer's step and its search together, as a program runs them -- rows in, attention with weights, logits, the choice, the cache behind its parents, now and
    then an eviction -- against the same in 64 bits: choices follow the kernel's logits, cache and weights the definition."""
    g = torch.Generator().manual_seed(beams)
    batch, heads, ctx, vocab, keep = 2, 2, 96, 500, 48
    n = batch * beams
    cache, w = BlockCache(n, ctx, heads, dim), torch.zeros(n, heads, ctx, device="cuda")
    prompt = torch.randn(batch, 50, heads, dim, generator=g).to(BF16)
    both = prompt.repeat_interleave(beams, 0)
    cache.append(both.cuda(), both.flip(1).cuda(), torch.zeros(n, dtype=I32, device="cuda"))
    values = [U.held(cache.k.cpu(), cache.k_exp.cpu()), U.held(cache.v.cpu(), cache.v_exp.cpu())]
    exps = [(e.cpu().int() - 127) for e in (cache.k_exp, cache.v_exp)]
    wref = torch.zeros(n, heads, ctx, dtype=torch.float64)
    out_w = torch.randn(heads * group * dim, vocab, generator=g) * 0.3
    emb = torch.randn(vocab, (heads * group + 2 * heads) * dim, generator=g)
    length = torch.full((n,), 50, dtype=I32, device="cuda")
    scores, ended = torch.full((batch, beams), -math.inf), torch.zeros(batch, beams, dtype=I32)
    scores[:, 0] = 0
    gs, ge = scores.cuda(), ended.cuda()
    tokens = torch.arange(batch).repeat_interleave(beams)
    for step in range(20):
        rows = emb[tokens].view(n, 1, heads * group + 2 * heads, dim).to(BF16)
        q, k, v = rows.split([heads * group, heads, heads], 2)
        dev = rows.cuda()
        cache.append(dev[:, :, heads * group : heads * group + heads], dev[:, :, heads * group + heads :], length)
        length += 1
        o = cache.attention(dev[:, :, : heads * group], length, weights=w, max_len=ctx)
        lens = length.tolist()
        for i in range(n):
            for h in range(heads):
                for x, vals, ex in ((k, values[0], exps[0]), (v, values[1], exps[1])):
                    e = ex[i, h].tolist()
                    U.append(vals[i, h], e, x[i, :, h], lens[i] - 1, 1)
                    ex[i, h] = torch.tensor(e)
            want, wt, size, most, mass = U.attention(q[i], values[0][i], values[1][i], lens[i], lens[i] - 1, 0, dim**-0.5)
            tol = U.attention_tolerance(want, size, most, mass, dim, lens[i], float(values[1][i, :, : lens[i]].abs().max()))
            assert bool(((o[i].cpu().double() - want).abs() <= tol).all()), f"step {step}, sequence {i}"
            wref[i] += wt
            near = (w[i, :, : lens[i]].cpu().double() - wref[i, :, : lens[i]]).abs()
            assert bool((near <= (step + 1) * (U.weights_tolerance(torch.ones(()), most, mass, dim, group) + 2.0**-20)).all())
        logits = (o.view(n, -1).float() @ out_w.cuda())
        choice = select_beams(logits, gs, ended=ge, end_id=7)
        for b in range(batch):
            want = U.beams(logits[b * beams : (b + 1) * beams].cpu(), gs[b].cpu(), ge[b].cpu(), 7, -1, None)
            assert choice.tokens[b].tolist() == [c[0] for c in want] and choice.parents[b].tolist() == [c[1] for c in want] and choice.ended[b].tolist() == [c[3] for c in want]
        reorder_states([cache.k, cache.v, cache.k_exp, cache.v_exp, w, length], choice.parents)
        slots = (choice.parents.cpu() + torch.arange(batch)[:, None] * beams).view(-1)
        values, exps, wref = [x[slots] for x in values], [x[slots] for x in exps], wref[slots]
        gs, ge, tokens = choice.scores, choice.ended, choice.tokens.cpu().view(-1).long()
        if step in (6, 13):
            had, lens = w.cpu(), length.tolist()
            kept, new = cache.evict(w, length, keep, first=2, recent=8)
            length.copy_(new)
            for i in range(n):
                for h in range(heads):
                    rows_ = U.kept_rows(had[i, h].tolist(), lens[i], keep, 2, 8)
                    assert kept[i, h, : len(rows_)].tolist() == rows_
                    wref[i, h, : len(rows_)] = wref[i, h][rows_]
                    for vals, ex in zip(values, exps):
                        took = vals[i, h][rows_]
                        for b0 in range(0, len(rows_), U.BLOCK):
                            part = took[b0 : b0 + U.BLOCK]
                            e = U.exponent(U.finite_top(part))
                            ex[i, h, b0 // U.BLOCK] = e
                            vals[i, h, b0 : b0 + len(part)] = U.e4m3(part * 2.0**-e) * 2.0**e
        gk, gv = cache.read(None, ctx, kv_len=length)
        for i in range(n):
            m = int(length[i])
            assert torch.equal(gk[i, :, :m].cpu().double(), values[0][i, :, :m]) and torch.equal(gv[i, :, :m].cpu().double(), values[1][i, :, :m])
