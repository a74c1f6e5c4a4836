"""Outputs that would be written over their inputs or over one another: refused before anything is launched.  No GPU."""
import ctypes as C

import pytest

from moondream_amd import _lib

from test_blocks_cpu import AT, GB, attention_args, cache

INVALID, WORKSPACE = 1, 3


def attend(**kw):
    """The status of a call whose workspace is missing: WORKSPACE where all else is as it has to be (nothing is launched either way)."""
    long = cache(ctx=1 << 15)
    return _lib.load().md_kv8_attention(C.byref(long), C.byref(attention_args(**{**dict(n_heads=4, q_len=3, batch=2, q_bs=3 * 256, q_ts=256, q_hs=64, o_bs=3 * 256, o_ts=256, o_hs=64), **kw})), None)


@pytest.mark.parametrize("weights", [None, AT + 20 * GB])
@pytest.mark.parametrize("bad", [dict(o=AT + 128), dict(o=AT + 512), dict(o=AT + 2 * 3 * 256), dict(o=AT - 64, q_bs=3 * 512, q_ts=512, q_hs=128, o_bs=3 * 512, o_ts=512, o_hs=128),
                                 dict(o=AT, o_ts=64, o_hs=3 * 64), dict(o=AT, o_bs=4 * 256), dict(o_ts=0), dict(o_hs=0), dict(o_bs=0), dict(o_hs=32), dict(o_ts=128),
                                 dict(o_bs=256), dict(o=AT + 1024, q_ts=512, q_bs=3 * 512), dict(o=AT, o_ts=-256)], ids=str)
def test_attention_refuses_outputs_over_queries_or_one_another(weights, bad):
    assert attend(weights=weights, **bad) == INVALID


@pytest.mark.parametrize("weights", [None, AT + 20 * GB])
@pytest.mark.parametrize("good", [dict(), dict(o=AT + 2 * 2 * 3 * 256), dict(o=AT + 512, q_bs=3 * 512, q_ts=512, o_bs=3 * 512, o_ts=512),  # another part of the same rows
                                  dict(o=AT + 128, q_bs=3 * 512, q_ts=512, q_hs=128, o_bs=3 * 512, o_ts=512, o_hs=128), dict(q_bs=0), dict(q_ts=0, q_hs=0),
                                  dict(o_bs=64, o_hs=128, o_ts=512), dict(batch=1, o_bs=0), dict(q_len=1, o_ts=0, o=AT + 1024, o_bs=256 * 3),
                                  dict(o=AT + 256, q_len=1, q_ts=0, o_ts=8, batch=1, q_bs=8, o_bs=0, n_heads=2)], ids=str)
def test_attention_takes_outputs_between_queries(weights, good):
    assert attend(weights=weights, **good) == WORKSPACE


def test_attention_in_the_queries_place():
    assert attend(o=AT) == WORKSPACE and attend(o=AT, weights=AT + 20 * GB) == INVALID
    assert attend(o=AT, q_len=1, o_ts=8) == WORKSPACE  # (a stride that no element is apart by)
