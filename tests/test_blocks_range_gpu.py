"""Attention over long caches on the GPU: a first row that takes most of the weight, blocks that all matter, one sequence alone and in a batch, queries that are no numbers."""
import math

import pytest
import torch

from moondream_amd.block_cache import BlockCache

import blocks_range as R
import blocks_util as U

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def one_slot(k, v, heads):
    """A cache of one slot whose heads all hold the same rows."""
    n, dim = k.shape
    c = BlockCache(1, n, heads, dim)
    c.append(*(x.cuda()[None, :, None].expand(1, n, heads, dim) for x in (k, v)), ints([0]))
    return c


def held(c, n):
    """Head 0's keys and values in 64 bits, and the values' scale exponents, row by row."""
    k, v = U.held(c.k[0, 0].cpu(), c.k_exp[0, 0].cpu()), U.held(c.v[0, 0].cpu(), c.v_exp[0, 0].cpu())
    return k[:n], v[:n], (c.v_exp[0, 0].cpu().int() - 127).repeat_interleave(U.BLOCK)[:n]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("share, size, outlier", R.SINKS)
@pytest.mark.parametrize("batch, tokens", [(1, 1), (34, 1), (3, 1), (17, 40), (6, 300)])  # keys over workgroups or not; 16 and 32 columns a wave
def test_a_first_row_that_takes_most_of_the_weight(dim, share, size, outlier, batch, tokens):
    n, heads = 32768, 32
    c = one_slot(*R.sink(n, dim, share, size, outlier, 3), heads)
    k, v, e = held(c, n)
    q = torch.randn(batch, tokens, heads, dim, generator=torch.Generator().manual_seed(batch + tokens))
    q[..., 0] = 8.0
    q = q.to(BF16)
    got = c.attention(q.cuda(), ints([n] * batch), slot=ints([0] * batch)).cpu().double()
    for b, h in ((0, 0), (batch - 1, heads - 1)):
        t = slice(max(0, tokens - 20), tokens)
        _, _, o, tol = R.one_head(q[b, t, h], k, v, e, dim**-0.5, n - tokens + t.start)
        worst = float(((got[b, t, h] - o).abs() / tol).max())
        assert worst <= 1, f"sequence {b}, head {h}: {worst} times the tolerance"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", R.LENGTHS)
@pytest.mark.parametrize("batch, group, tokens", [(1, 1, 1), (1, 4, 1), (40, 1, 1), (1, 1, 3), (2, 8, 4), (1, 1, 40), (20, 2, 40)])
def test_every_block_of_a_long_cache_reaches_the_output(dim, n, batch, group, tokens):
    heads = 32 if batch > 2 else 2
    c = one_slot(*R.marked(n, dim, n), heads)
    k, v, e = held(c, n)
    q = (torch.randn(batch, tokens, heads * group, dim, generator=torch.Generator().manual_seed(n + batch)) * 0.1).to(BF16)
    got = c.attention(q.cuda(), ints([n] * batch), slot=ints([0] * batch)).cpu().double()
    for b, h in ((0, 0), (batch - 1, heads * group - 1)):
        _, _, o, tol = R.one_head(q[b, :, h], k, v, e, dim**-0.5, n - tokens)
        worst = float(((got[b, :, h] - o).abs() / tol).max())
        assert worst <= 1, f"sequence {b}, head {h}: {worst} times the tolerance"


@pytest.mark.parametrize("dim, group, tokens", [(64, 1, 1), (128, 8, 1), (64, 4, 3), (128, 1, 40), (64, 2, 200)])
def test_a_sequence_alone_and_in_a_batch(dim, group, tokens):
    """The launch is cut by the counts of the call: sums may come in another order, and each is as near to 64 bits as it has to be.  The weights too."""
    n, heads, batch = 2500, 4, 70
    c = one_slot(*R.marked(n, dim, 1), heads)
    more = BlockCache.of(*(t.expand(batch, *t.shape[1:]).contiguous() for t in (c.k, c.v, c.k_exp, c.v_exp)))
    k, v, e = held(c, n)
    q = (torch.randn(1, tokens, heads * group, dim, generator=torch.Generator().manual_seed(7)) * 0.3).to(BF16)
    w1, wb = torch.zeros(1, heads, c.ctx, device="cuda"), torch.zeros(batch, heads, c.ctx, device="cuda")
    alone = c.attention(q.cuda(), ints([n]), weights=w1, decay=0.0)
    among = more.attention(q.cuda().expand(batch, -1, -1, -1), ints([n] * batch), weights=wb, decay=0.0)
    assert bool((among == among[:1]).all()) and bool((wb == wb[:1]).all())
    h = heads * group - 1
    p, _, o, tol = R.one_head(q[0, :, h], k, v, e, dim**-0.5, n - tokens)
    for got in (alone, among):
        assert bool(((got[0, :, h].cpu().double() - o).abs() <= tol).all())
    want, most, mass = torch.zeros(n, dtype=torch.float64), 0.0, 0.0
    for j in range(group):
        x = q[0, :, (heads - 1) * group + j].double()
        want += R.one_head(x, k, v, e, dim**-0.5, n - tokens)[0].sum(0)
        most, mass = max(most, float((x @ k.T).abs().max() * dim**-0.5)), max(mass, float((x.abs() @ k.abs().T).max() * dim**-0.5))
    for got in (w1, wb):
        assert bool(((got[0, heads - 1, :n].cpu().double() - want).abs() <= U.weights_tolerance(want, most, mass, dim, tokens * group)).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens, group", [(4, 1), (9, 2), (100, 1), (300, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_is_no_number_leaves_rows_alone_that_it_does_not_see(dim, tokens, group, bad):
    g = torch.Generator().manual_seed(tokens)
    n, heads = tokens + 45, 2
    c = BlockCache(1, n, heads, dim)
    x = torch.randn(1, n, heads, dim, generator=g).to(BF16).cuda()
    c.append(x, x, ints([0]))
    q = torch.randn(1, tokens, heads * group, dim, generator=g).to(BF16).cuda()
    sick, well = q.clone(), q.clone()
    at = tokens // 2
    sick[0, at, 0, 5], well[0, at, 0] = bad, 0.0
    w, clean = (torch.zeros(1, heads, c.ctx, device="cuda") for _ in range(2))
    c.attention(sick, ints([n]), weights=w)
    c.attention(well, ints([n]), weights=clean)
    seen = n - tokens + at + 1
    assert bool(torch.isnan(w[0, 0, :seen]).any()) and torch.equal(w[0, 0, seen:], clean[0, 0, seen:]) and torch.equal(w[0, 1], clean[0, 1])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, tokens", [(1, 1), (40, 1), (2, 3), (2, 40), (20, 200)])
def test_scores_of_millions_stay_finite(dim, batch, tokens):
    """Scores of 2^24 and more in units of log2, which fp32 holds to whole numbers: outputs are still means of values."""
    g = torch.Generator().manual_seed(dim + tokens)
    n, heads = 4096, 32
    k, v = torch.zeros(n, dim), torch.randn(n, dim, generator=g)
    k[:, 0] = 4096.0
    k[:, 1] = torch.arange(n) // U.BLOCK * 8.0  # block by block a little more, about as much as a running maximum may fall behind
    c = one_slot(k.to(BF16), v.to(BF16), heads)
    top = float(c.read(None, n)[1].abs().max())
    q = torch.zeros(batch, tokens, heads, dim)
    q[..., 0] = torch.randint(3000, 8192, (batch, tokens, heads), generator=g).float()
    q[..., 1] = torch.rand(batch, tokens, heads, generator=g) * 2
    got = c.attention(q.to(BF16).cuda(), ints([n] * batch), slot=ints([0] * batch), scale=1.0).float()
    assert bool(torch.isfinite(got).all())
    # fp16 weights are off by 2^-11, sums over keys by n * 2^-23, the output by 2^-8
    assert float(got.abs().max()) <= top * (1 + 2.0**-11 + n * 2.0**-23) * (1 + 2.0**-8)
