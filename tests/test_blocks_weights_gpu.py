"""Weights of a few tokens on the GPU, from kept scores and from scores made again."""
import pytest
import torch

from test_blocks_gpu import attend, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim, group, tokens", [(64, 1, 12), (64, 13, 1), (64, 4, 4), (64, 4, 8), (128, 8, 3), (128, 5, 5), (128, 26, 1), (128, 1, 32), (64, 1, 1)])
@pytest.mark.parametrize("batch, kv_heads, length", [(3, 2, 200), (5, 1, 3001), (2, 8, 700)])
def test_weights_from_kept_scores_and_from_keys_again(dim, group, tokens, batch, kv_heads, length):
    g = torch.Generator().manual_seed(dim + group + length)
    lens = [max(0, length - 97 * i) for i in range(batch - 1)] + [7]
    c, k, v = filled(g, batch, length, kv_heads, dim, junk=(lens, 0x7F))
    q = torch.randn(batch, tokens, kv_heads * group, dim, generator=g).to(torch.bfloat16)
    attend(c, k, v, q, lens, weights=True, decay=0.75)
    attend(c, k, v, q, lens, weights=True, decay=0.0, q_rows=[tokens // 2 + 1, 0, tokens, 1, tokens][:batch], prefix=50, max_len=length - 5)
    c, k, v = filled(g, batch, length, kv_heads, dim)  # (here every row of every slot may be seen)
    attend(c, k, v, q, lens, weights=True, slot=[(i + 1) % (batch + 1) for i in range(batch)], q_pos0=[3 * i - 1 for i in range(batch)])  # the last slot there is not


@pytest.mark.parametrize("dim, group, tokens, n", [(64, 4, 1, 9000), (128, 8, 1, 30000), (128, 4, 8, 9000), (64, 1, 200, 3000), (128, 2, 300, 4000)])
def test_weights_lean_to_no_side(dim, group, tokens, n):
    """Roundings are to the nearest; what may lean is the hardware's exponential (an ulp, 2^-23) against the sum's own, and the sum's reciprocal (2^-24): less than 2^-22 together.
    The scores' own roundings have either sign: over all rows and heads their mean is less than a quarter of that."""
    import blocks_util as U

    g = torch.Generator().manual_seed(n)
    heads = 4
    c, k, v = filled(g, 1, n, heads, dim)
    q = (torch.randn(1, tokens, heads * group, dim, generator=g) * 0.7).to(torch.bfloat16)
    w = torch.zeros(1, heads, c.ctx, device="cuda")
    c.attention(q.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), weights=w, decay=0.0)
    _, want, _, _, _ = U.attention(q[0], k[0], v[0], n, n - tokens, 0, dim**-0.5)
    off = (w[0, :, :n].cpu().double() / want[:, :n] - 1)[want[:, :n] > 1e-20]
    assert abs(float(off.mean())) < 2.0**-22, float(off.mean())


def test_an_output_of_one_sequence_or_token_may_have_any_stride_there():
    g = torch.Generator().manual_seed(3)
    c, _, _ = filled(g, 1, 64, 2, 64)
    q = torch.randn(1, 1, 4, 64, generator=g).to(torch.bfloat16).cuda()
    n = torch.tensor([60], dtype=torch.int32, device="cuda")
    out = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 4, 64), (0, 0, 64, 1))
    assert torch.equal(c.attention(q, n, out=out), c.attention(q, n))
    with pytest.raises(ValueError):
        c.attention(q, n, out=out[:, :, :1].expand(1, 1, 4, 64))
