"""The choice among beams whose logits are alike, in rows of every alignment: sums of exponentials follow the tokens, not the addresses, and are in 64 bits."""
import pytest
import torch

from moondream_amd.beams import select_beams

import blocks_util as U

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype, vocab", [(F32, 131075), (F32, 5001), (F32, 8191), (BF16, 8193), (BF16, 5001), (BF16, 51203), (F32, 4), (BF16, 9)])
@pytest.mark.parametrize("batch, beams", [(1, 2), (2, 4), (7, 5), (3, 16)])
def test_equal_rows_are_ties(dtype, vocab, batch, beams):
    g = torch.Generator().manual_seed(vocab + beams)
    for draw in range(4):
        row = (torch.randn(batch, 1, vocab, generator=g) * 3).to(dtype)
        if draw % 2:
            row[:, 0, -1] = row.float().amax(-1)[:, 0].to(dtype) + 1  # the best token is the last one
        logits = row.expand(batch, beams, vocab).reshape(batch * beams, vocab).cuda()
        got = select_beams(logits, torch.full((batch, beams), -1.5, device="cuda"))
        best = torch.sort(row[:, 0].double(), dim=-1, descending=True, stable=True)
        for b in range(batch):  # rank by rank: all beams' best token, the lowest beam first
            order = [(float(v), k, int(t)) for t, v in zip(best.indices[b, :beams], best.values[b, :beams]) for k in range(beams)]
            order.sort(key=lambda c: (-c[0], c[1], c[2]))
            assert got.parents[b].tolist() == [c[1] for c in order[:beams]] and got.tokens[b].tolist() == [c[2] for c in order[:beams]], draw
            assert len({x for x, c in zip(got.scores[b].tolist(), order) if c[0] == order[0][0]}) == 1


@pytest.mark.parametrize("dtype, vocab", [(F32, 131075), (F32, 5001), (BF16, 51203)])
def test_sums_are_in_64_bits(dtype, vocab):
    """Beams whose sums differ by some parts in 10^10: one rare token a little more likely in the lower beam, whose totals are the smaller ones for it."""
    g = torch.Generator().manual_seed(vocab)
    for draw in range(12):
        row = (torch.randn(1, vocab, generator=g) * 3).to(dtype)
        top = float(row.float().max())
        logits = row.repeat(2, 1)
        rare = int(torch.randint(0, vocab, (1,), generator=g))
        logits[:, rare] = top - 20.0
        logits[draw % 2, rare] = top - 19.0
        scores = torch.zeros(1, 2)
        want = U.beams(logits, scores[0], None, -1, -1, None)
        got = select_beams(logits.cuda(), scores.cuda())
        assert got.parents[0].tolist() == [w[1] for w in want] and got.tokens[0].tolist() == [w[0] for w in want]
        assert want[0][1] == 1 - draw % 2
        for x, w in zip(got.scores[0].tolist(), want):
            assert abs(x - w[2]) <= abs(w[2]) * 2.0**-24 + 1e-12  # one rounding to fp32; sums in 64 bits


def test_sums_of_far_apart_and_of_extreme_logits():
    far = torch.tensor([[0.0, -80.0, -104.0, -500.0, -3e38], [3e38, 3e38, -3e38, 0.0, 1.0], [1e-40, -1e-40, 0.0, -0.0, 1e-45], [-3.4e38] * 5])
    scores = torch.tensor([[-1.0, -2.0], [-3.0, -4.0]])
    got = select_beams(far.cuda(), scores.cuda())
    for b in range(2):
        want = U.beams(far[2 * b : 2 * b + 2], scores[b], None, -1, -1, None)
        assert got.tokens[b].tolist() == [w[0] for w in want] and got.parents[b].tolist() == [w[1] for w in want]
        for x, w in zip(got.scores[b].tolist(), want):
            assert abs(x - w[2]) <= abs(w[2]) * 2.0**-24 + 1e-12


@pytest.mark.parametrize("beams", [2, 5])
def test_states_between_one_another(beams):
    """From one layer's part of a slab [slots, layers, ...] into another's, and from some rows of an answer to others: ranges that overlap, no byte in common."""
    from moondream_amd.beams import reorder_states

    g = torch.Generator().manual_seed(beams)
    n = 3 * beams
    slab = torch.randn(n, 3, 4, 50, 16, generator=g).cuda()
    parents = torch.randint(0, beams, (3, beams), generator=g)
    slots = (parents + torch.arange(3)[:, None] * beams).view(-1).cuda()
    want = slab.clone()
    want[:, 2] = slab[slots, 1]
    want[:, 0, :, 30:41] = slab[slots, 0, :, 3:14]
    reorder_states([slab[:, 1]], parents.to(torch.int32).cuda(), into=[slab[:, 2]])
    reorder_states([slab[:, 0, :, 3:14]], parents.to(torch.int32).cuda(), into=[slab[:, 0, :, 30:41]])
    assert torch.equal(slab, want)


def test_a_state_twice_and_two_states_in_each_others_place_are_refused():
    from moondream_amd import _lib
    from moondream_amd.beams import reorder_states

    a, b = torch.arange(16.0, device="cuda").view(4, 4), torch.ones(4, 4, device="cuda")
    parents = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda")
    for states, into in (([a, b, a], None), ([a, b], [b, a]), ([a, b], [torch.zeros_like(a)] * 2)):
        with pytest.raises(_lib.MoondreamHipError):
            reorder_states(states, parents, into=into)
    assert torch.equal(a, torch.arange(16.0, device="cuda").view(4, 4)) and bool((b == 1).all())
    both = [torch.zeros_like(a), torch.zeros_like(a)]
    reorder_states([a, a], parents, into=both)  # one that is read twice is fine
    assert torch.equal(both[0], a[[1, 0, 3, 3]]) and torch.equal(both[1], both[0])
