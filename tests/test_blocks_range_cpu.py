"""The bound on long caches' outputs sees what it is for: mistakes planted in the oracle, on the CPU."""
import pytest
import torch

import blocks_range as R
import blocks_util as U


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", R.LENGTHS)
def test_every_block_of_a_long_cache_matters(dim, n):
    k, v = R.marked(n, dim, n)
    (k, _), (v, e) = R.held_rows(k), R.held_rows(v)
    q = torch.randn(3, dim, generator=torch.Generator().manual_seed(1)) * 0.1
    p, _, o, tol = R.one_head(q.to(torch.bfloat16), k, v, e, dim**-0.5)
    pad = -n % U.BLOCK
    part = torch.nn.functional.pad(p[..., None] * v, (0, 0, 0, pad)).view(3, -1, U.BLOCK, dim)
    for lost in (part.sum(2), (part - part.roll(1, 2)).sum(2) + (part - part.roll(1, -1)).sum(2)):  # a block left out; its coordinates moved by one
        assert float(((lost.abs() / tol[:, None]).amax(-1)).min()) > 2


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("share, size, outlier", R.SINKS)
def test_weights_that_fp16_would_lose_matter(dim, share, size, outlier):
    """The largest scaled weight at 1 instead of 2^7: fp16 drops or roughens the many small ones, and the bound shows it."""
    n = 32768
    k, v = R.sink(n, dim, share, size, outlier, 3)
    (k, _), (v, e) = R.held_rows(k), R.held_rows(v)
    q = torch.randn(2, dim, generator=torch.Generator().manual_seed(2))
    q[:, 0] = 8.0
    p, y, o, tol = R.one_head(q.to(torch.bfloat16), k, v, e, dim**-0.5)
    assert abs(float(p[0, 0]) - share) < 0.2 * (1 - share) + 0.01
    unit = torch.exp2(e.double())
    for lift, within in ((0, False), (R.LIFT, True)):
        top = y.amax(-1, keepdim=True) * 2.0**-lift
        got = ((y / top).to(torch.float16).double() * top / unit) @ v
        worst = float(((got - o).abs() / tol).max())
        assert (worst <= 1) == within, (lift, worst)
