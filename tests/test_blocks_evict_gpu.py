"""Eviction on the GPU: which caches it goes between."""
import pytest
import torch

from moondream_amd.block_cache import BlockCache

from test_blocks_gpu import filled, ints

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
