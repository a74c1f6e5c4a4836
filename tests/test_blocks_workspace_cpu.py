"""How much workspace attention asks for.  No GPU."""
import ctypes as C

import pytest

from moondream_amd import _lib

from test_blocks_cpu import AT, attention_args, cache


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group, tokens", [(1, 1), (4, 1), (1, 12), (13, 1), (1, 24), (25, 1), (1, 32), (8, 4), (4, 100)])
def test_weights_ask_for_less_than_half_the_cache(dim, group, tokens):
    """Beyond what the attention itself takes: kept scores, sums, shares."""
    lib, c = _lib.load(), cache(slots=64, ctx=1 << 15, kv_heads=32, dim=dim)
    a = attention_args(batch=64, n_heads=32 * group, q_len=tokens, q_hs=dim, o_hs=dim)
    bare = lib.md_kv8_attention_workspace_bytes(C.byref(c), C.byref(a))
    a.weights = AT
    need = lib.md_kv8_attention_workspace_bytes(C.byref(c), C.byref(a))
    assert bare < need and need - bare <= 2 * 64 * 32 * (1 << 15) * dim * 3 // 8 + (1 << 20) + 64 * 32 * group * tokens * 4
