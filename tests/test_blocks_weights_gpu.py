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
