"""States whose runs would be written over one another, and vocabularies past 32 bits: refused.  No GPU, nothing is launched."""
import ctypes as C

import pytest

from moondream_amd import _lib

from test_blocks_cpu import AT, beam_args, part


@pytest.mark.parametrize("bad", [dict(src_slot_stride=64, dst_slot_stride=64, src_seg_stride=64, dst_seg_stride=64), dict(dst_slot_stride=128), dict(outer=2, src_outer_stride=1024, dst_outer_stride=1024),
                                 dict(dst=AT, src_slot_stride=192, dst_slot_stride=192), dict(dst=AT + 256), dict(dst=AT + 32, src_seg_stride=128, dst_seg_stride=128, src_slot_stride=512, dst_slot_stride=512),
                                 dict(dst=AT + 64, src_seg_stride=128, dst_seg_stride=192, src_slot_stride=512, dst_slot_stride=768)], ids=str)
def test_reordering_refuses_runs_that_meet(bad):
    assert _lib.load().md_state_reorder(C.byref(part(**bad)), 1, AT, 2, 4, None) == 1


def test_a_vocabulary_that_32_bits_cannot_count_is_refused():
    lib = _lib.load()
    for vocab, ok in ((2**31 - 1, False), (2**31 - 8192, False), (2**31 - 8193, True)):
        assert (lib.md_beam_workspace_bytes(1, 2, vocab) > 0) == ok
        a = beam_args(batch=1, beams=2, vocab=vocab, ld=2**31, workspace=None)  # (a missing workspace: nothing is launched)
        assert lib.md_beam_select(C.byref(a), None) == (3 if ok else 1)


def test_pieces_that_write_what_another_moves_are_refused():
    lib, there = _lib.load(), 1 << 33
    apart = dict(src=there, dst=there + AT)
    for pieces in ([part(), part()], [part(src=AT, dst=AT), part(src=AT, dst=AT)], [part(), part(src=part().dst, dst=part().src)], [part(), part(**apart), part(src=part().dst, dst=2 * there)],
                   [part(**apart), part(), part(src=2 * there, dst=part().dst)]):
        assert lib.md_state_reorder((_lib.MdStatePart * len(pieces))(*pieces), len(pieces), AT, 2, 4, None) == 1
