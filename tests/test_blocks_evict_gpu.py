"""Eviction on the GPU: which caches it goes between."""
import pytest
import torch

from moondream_amd.block_cache import BlockCache

from test_blocks_gpu import filled, ints, random_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("of", ["itself", "another over its tensors"])
def test_a_cache_into_itself_is_refused(of):
    """It would run in place and leave the weights behind: in place is without into."""
    c, _, _ = filled(torch.Generator().manual_seed(1), 2, 96, 2, 64)
    into = c if of == "itself" else BlockCache.of(c.k, c.v, c.k_exp, c.v_exp)
    w = torch.rand(2, 2, 96, device="cuda")
    before = c.k.clone(), w.clone()
    for into_weights in (None, w, torch.zeros_like(w)):
        with pytest.raises(ValueError):
            c.evict(w, ints([96, 90]), 40, into=into, into_weights=into_weights)
    assert torch.equal(before[0], c.k) and torch.equal(before[1], w)


@pytest.mark.parametrize("keep", [40, 64])
def test_from_one_layer_s_slots_into_another_s_between_them(keep):
    """Slabs [slots, layers, ...]: the layers' slots lie between one another and share no byte."""
    g = torch.Generator().manual_seed(3)
    slots, heads, ctx, dim = 3, 2, 96, 64
    whole = [torch.zeros(slots, 3, heads, ctx, dim, dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.full((slots, 3, heads, ctx // 32), 87, dtype=torch.uint8, device="cuda") for _ in range(2)]
    layers = [BlockCache.of(*(t[:, i] for t in whole)) for i in range(3)]
    x, y = (random_rows(g, slots, ctx, heads, dim).cuda() for _ in range(2))
    alone, into = BlockCache(slots, ctx, heads, dim), BlockCache(slots, ctx, heads, dim)
    for c in (layers[1], alone):
        c.append(x, y, ints([0] * slots))
    w = torch.rand(slots, heads, ctx, generator=g).cuda()
    w1, w2 = torch.zeros_like(w), torch.zeros_like(w)
    lens = ints([96, 50, 30])
    before = [t[:, 1].clone() for t in whole]
    for to, out in ((layers[2], w1), (layers[0], w1)):
        kept, n = layers[1].evict(w, lens, keep, recent=8, into=to, into_weights=out)
        kept2, n2 = alone.evict(w, lens, keep, recent=8, into=into, into_weights=w2)
        assert torch.equal(kept, kept2) and torch.equal(n, n2) and torch.equal(w1, w2)
        for a, b in zip(to.read(None, ctx, kv_len=n), into.read(None, ctx, kv_len=n)):
            assert torch.equal(a, b)
    assert all(torch.equal(t[:, 1], b) for t, b in zip(whole, before))


def test_caches_that_share_some_slots_are_refused():
    from moondream_amd._lib import MoondreamHipError

    c, _, _ = filled(torch.Generator().manual_seed(2), 4, 64, 2, 64)
    first, last = (BlockCache.of(*(t[s] for t in (c.k, c.v, c.k_exp, c.v_exp))) for s in (slice(0, 3), slice(1, 4)))
    w = torch.rand(3, 2, 64, device="cuda")
    even = BlockCache.of(*(t[::2] for t in (c.k, c.v, c.k_exp, c.v_exp)))
    odd = BlockCache.of(*(t[1::2] for t in (c.k, c.v, c.k_exp, c.v_exp)))
    before = c.k.clone()
    for a, b in ((first, last), (last, first), (first, even)):
        with pytest.raises((ValueError, MoondreamHipError)):
            a.evict(w[: a.slots].contiguous(), ints([64] * 2), 8, into=b)
    assert torch.equal(c.k, before)
    even.evict(w[:2].contiguous(), ints([64] * 2), 8, into=odd)
    assert torch.equal(c.k[::2], before[::2])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [1, 40])
def test_rows_that_come_after_an_eviction_begin_without_weight(dim, tokens):
    """Steps as a program runs them: rows in, attention, an eviction in place, rows in where evicted ones were; then a new sequence in a used slot."""
    import blocks_util as U

    g = torch.Generator().manual_seed(dim + tokens)
    heads, ctx = 2, 160
    c, w = BlockCache(3, ctx, heads, dim), torch.zeros(3, heads, ctx, device="cuda")
    slot, length = ints([2, 0]), ints([0, 0])

    def step(length):
        x, y, q = (random_rows(g, 2, tokens, heads, dim, spread=0.5).cuda() for _ in range(3))
        c.append(x, y, length, slot=slot, weights=w)
        length = length + tokens
        c.attention(q, length, slot=slot, weights=w)
        return q.cpu(), length

    for _ in range(100 // tokens):
        _, length = step(length)
    had = w.cpu()
    kept, length = c.evict(w, length, 20, recent=4, slot=slot)
    assert length.tolist() == [20, 20] and bool((w[2, :, 20 : 20 + tokens] != 0).any())
    for fresh in (False, True):
        if fresh:
            length = ints([0, 0])
        before = torch.zeros(3, heads, ctx, dtype=torch.float64) if fresh else w.cpu().double()
        start = int(length[0])
        q, length = step(length)
        k, v = (U.held(t.cpu(), e.cpu()) for t, e in ((c.k, c.k_exp), (c.v, c.v_exp)))
        for b, s in enumerate((2, 0)):
            n = start + tokens
            _, want, _, most, mass = U.attention(q[b], k[s], v[s], n, start, 0, dim**-0.5)
            want[:, :start] += before[s, :, :start]
            near = (w[s, :, :n].cpu().double() - want[:, :n]).abs()
            assert bool((near <= U.weights_tolerance(want[:, :n], most, mass, dim, tokens) + want[:, :n] * 2.0**-23).all())
    assert not bool(w[1].any()) and bool((had[0] != 0).any())


def test_the_weights_of_rows_that_are_not_new_stay():
    c, w = BlockCache(4, 96, 3, 64), torch.ones(4, 3, 96, device="cuda")
    x = torch.ones(5, 40, 3, 64, dtype=torch.bfloat16, device="cuda")
    c.append(x, x, ints([10, 90, 31, -1, 0]), new=ints([40, 9, 0, 5, 33]), slot=ints([3, 0, 1, 1, 4]), weights=w)
    want = torch.ones(4, 3, 96)
    want[3, :, 10:50] = 0
    want[0, :, 90:] = 0
    assert torch.equal(w.cpu(), want)
    for bad in (w[:3], w.double(), w[:, :, :95], w.cpu()):
        with pytest.raises(ValueError):
            c.append(x, x, ints([0] * 5), slot=ints([3, 0, 1, 1, 4]), weights=bad)
