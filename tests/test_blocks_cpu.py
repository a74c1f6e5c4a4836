"""The block cache's and the beams' entry points: structs, refusals (nothing is launched), and the 64-bit oracle's own numbers.  No GPU."""
import ctypes as C
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from moondream_amd import _lib
from moondream_amd.beams import _runs, reorder_states, select_beams
from moondream_amd.block_cache import BlockCache

import blocks_util as U

AT = 4096  # an address that nothing reads: refused before that
GB = 1 << 30


def cache(at=AT, slots=4, ctx=64, kv_heads=2, dim=64, **kw):
    c = _lib.MdKv8Cache(at, at + GB, at + 2 * GB, at + 3 * GB, kv_heads * ctx * dim, kv_heads * ctx // 32, slots, ctx, kv_heads, dim)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(head_dim=72), dict(head_dim=32), dict(ctx=65), dict(ctx=0), dict(k=None), dict(v_exp=None), dict(slots=0), dict(kv_heads=0),
              dict(slot_stride=64), dict(slot_stride=2 * 64 * 64 + 8), dict(exp_stride=3), dict(k=AT + 8)]


def append(c, k=AT, ks=(256, 128, 64), v=AT, slot=None, row0=AT, new=None, batch=2, tokens=2):
    return _lib.load().md_kv8_append(C.byref(c) if c is not None else None, k, *ks, v, *ks, slot, row0, new, batch, tokens, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_no_entry_point_takes_a_broken_cache(bad):
    lib, c = _lib.load(), cache(**bad)
    assert append(c) == 1
    assert lib.md_kv8_read(C.byref(c), None, None, None, 1, 1, AT, AT, None) == 1
    assert lib.md_kv8_attention(C.byref(c), C.byref(attention_args()), None) == 1
    assert lib.md_kv8_attention_workspace_bytes(C.byref(c), C.byref(attention_args())) == 0
    for pair in ((c, cache(AT + 8 * GB)), (cache(AT + 8 * GB), c), (c, c)):
        assert lib.md_kv8_evict(C.byref(pair[0]), C.byref(pair[1]), C.byref(evict_args()), None) == 1


def test_append_and_read_refuse():
    lib, c = _lib.load(), cache()
    assert append(None) == 1
    for bad in (dict(k=None), dict(v=None), dict(row0=None), dict(batch=0), dict(tokens=0), dict(batch=5), dict(k=AT + 2), dict(ks=(256, 128, 65)), dict(ks=(4, 128, 64)),
                dict(batch=1 << 30, tokens=1 << 30, slot=AT)):
        assert append(c, **bad) == 1, bad
    ref = C.byref(c)
    for bad in ((None, None, None, 0, 1, AT, AT), (None, None, None, 5, 1, AT, AT), (None, None, None, 1, 0, AT, AT), (None, None, None, 1, 1, None, AT),
                (None, None, None, 1, 1, AT, AT + 8)):
        assert lib.md_kv8_read(ref, *bad, None) == 1, bad


def attention_args(**kw):
    a = _lib.MdKv8AttnArgs(AT, 256, 128, 64, AT + 5 * GB, 256, 128, 64, 2, 4, 1, None, None, None, AT, 0, 0, 0.125, 1.0, None, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(q=None), dict(o=None), dict(kv_len=None), dict(batch=0), dict(batch=5), dict(batch=70000, slot=AT), dict(q_len=0), dict(q_len=1 << 23),
                                 dict(n_heads=0), dict(n_heads=3), dict(max_len=-1), dict(prefix_len=-1), dict(q_ts=4), dict(o_hs=68), dict(q=AT + 4), dict(scale=math.nan),
                                 dict(scale=math.inf), dict(weights=AT, decay=-1.0), dict(weights=AT, decay=math.inf), dict(weights=AT, decay=math.nan), dict(weights=AT, o=AT), dict(n_heads=1 << 18, q_len=16)], ids=str)
def test_attention_refuses(bad):
    assert _lib.load().md_kv8_attention(C.byref(cache()), C.byref(attention_args(workspace=AT, workspace_bytes=GB, **bad)), None) == 1


def test_attention_names_the_workspace_that_it_needs():
    lib, long = _lib.load(), cache(ctx=1 << 15)
    a = attention_args(weights=AT)
    need = lib.md_kv8_attention_workspace_bytes(C.byref(long), C.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = AT, need - 1
    assert lib.md_kv8_attention(C.byref(long), C.byref(a), None) == 3
    a.workspace, a.workspace_bytes = None, need
    assert lib.md_kv8_attention(C.byref(long), C.byref(a), None) == 3
    a.workspace = AT + 4
    assert lib.md_kv8_attention(C.byref(long), C.byref(a), None) == 1


def evict_args(**kw):
    a = _lib.MdKv8EvictArgs(AT + 30 * GB, None, None, AT, AT, AT, 2, 32, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(weights=None), dict(kv_len=None), dict(len_out=None), dict(kept=None), dict(batch=0), dict(batch=5), dict(keep=0), dict(keep=65),
                                 dict(first=-1), dict(recent=-1), dict(first=20, recent=13), dict(first=2**31 - 1, recent=2**31 - 1)], ids=str)
def test_evict_refuses(bad):
    lib, a = _lib.load(), evict_args(**bad)
    assert lib.md_kv8_evict(C.byref(cache()), C.byref(cache(AT + 8 * GB)), C.byref(a), None) == 1
    assert lib.md_kv8_evict(C.byref(cache()), C.byref(cache()), C.byref(a), None) == 1


def test_evict_refuses_caches_that_share_part_of_their_memory():
    lib = _lib.load()
    assert lib.md_kv8_evict(C.byref(cache()), C.byref(cache(ctx=32, slot_stride=2 * 32 * 64, exp_stride=2)), C.byref(evict_args()), None) == 1  # same codes, other layout
    other = cache(AT + 8 * GB)
    other.k = AT + 64  # overlaps
    assert lib.md_kv8_evict(C.byref(cache()), C.byref(other), C.byref(evict_args()), None) == 1
    other = cache(AT + 8 * GB)
    other.v_exp = cache().k_exp
    assert lib.md_kv8_evict(C.byref(cache()), C.byref(other), C.byref(evict_args()), None) == 1
    for c in (cache(AT + 8 * GB, kv_heads=1, slot_stride=2 * 64 * 64), cache(AT + 8 * GB, dim=128)):
        assert lib.md_kv8_evict(C.byref(cache()), C.byref(c), C.byref(evict_args()), None) == 1
    a = evict_args(weights_out=AT + 30 * GB + 64)
    assert lib.md_kv8_evict(C.byref(cache()), C.byref(cache(AT + 8 * GB)), C.byref(a), None) == 1


def beam_args(**kw):
    a = _lib.MdBeamArgs(AT, 100, _lib.MD_DTYPE_F32, 2, 4, 100, -1, 0, AT, AT, None, AT, AT, AT, AT, AT, GB)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(logits=None), dict(scores=None), dict(tokens=None), dict(parents=None), dict(scores_out=None), dict(batch=0), dict(beams=1), dict(beams=17),
                                 dict(vocab=0), dict(ld=99), dict(dtype=2), dict(end_id=100), dict(end_id=-1), dict(logits=AT + 2), dict(batch=20000), dict(workspace=AT + 8)], ids=str)
def test_beam_choice_refuses(bad):
    assert _lib.load().md_beam_select(C.byref(beam_args(**bad)), None) == 1


def test_beam_choice_names_the_workspace_that_it_needs():
    lib = _lib.load()
    need = lib.md_beam_workspace_bytes(2, 4, 100)
    assert need > 0 and lib.md_beam_workspace_bytes(2, 1, 100) == lib.md_beam_workspace_bytes(0, 2, 100) == lib.md_beam_workspace_bytes(1, 17, 100) == 0
    assert lib.md_beam_select(C.byref(beam_args(workspace_bytes=need - 1)), None) == 3
    assert lib.md_beam_select(C.byref(beam_args(workspace=None)), None) == 3
    assert lib.md_beam_select(None, None) == 1


def part(**kw):
    p = _lib.MdStatePart(AT, AT + GB, 256, 256, 0, 0, 64, 64, 64, 1, 4)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad", [dict(src=None), dict(dst=None), dict(seg_bytes=0), dict(outer=0), dict(segs=0), dict(src_slot_stride=-256), dict(dst_seg_stride=32),
                                 dict(dst_slot_stride=0), dict(outer=2), dict(dst=AT + 64), dict(dst=AT, dst_slot_stride=512), dict(dst=AT, dst_seg_stride=128),
                                 dict(seg_bytes=1 << 40, dst_seg_stride=1 << 40, dst_slot_stride=1 << 50, dst=1 << 55)], ids=str)
def test_reordering_refuses(bad):
    lib = _lib.load()
    assert lib.md_state_reorder(C.byref(part(**bad)), 1, AT, 2, 4, None) == 1
    both = (_lib.MdStatePart * 2)(part(), part(**bad))  # one bad piece among good ones: nothing is moved
    assert lib.md_state_reorder(both, 2, AT, 2, 4, None) == 1


def test_reordering_refuses_its_numbers():
    lib = _lib.load()
    for n, parents, batch, beams in ((0, AT, 2, 4), (1, None, 2, 4), (1, AT, 0, 4), (1, AT, 2, 0), (1, AT, 2, 17), (1, AT, 70000, 2)):
        assert lib.md_state_reorder(C.byref(part()), n, parents, batch, beams, None) == 1
    assert lib.md_state_reorder(None, 1, AT, 2, 4, None) == 1


def test_struct_layouts_match_the_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "moondream_hip.h")
    pairs = {"md_kv8_cache": _lib.MdKv8Cache, "md_kv8_attn_args": _lib.MdKv8AttnArgs, "md_kv8_evict_args": _lib.MdKv8EvictArgs, "md_beam_args": _lib.MdBeamArgs,
             "md_state_part": _lib.MdStatePart}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {",
             'printf("%d %d %d %d\\n", MD_KV8_BLOCK, MD_MAX_BEAMS, MD_KV8_MIN_EXP, MD_KV8_MAX_EXP);']
    for name, cls in pairs.items():
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f[0]}));' for f in cls._fields_] + ['printf("\\n");']
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(src)], check=True)
    out = [[int(x) for x in line.split()] for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.strip().splitlines()]
    assert out[0] == [_lib.MD_KV8_BLOCK, _lib.MD_MAX_BEAMS, U.LOW, U.HIGH]
    for got, cls in zip(out[1:], pairs.values()):
        assert got == [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
        body = re.search(r"typedef struct \{((?:(?!typedef struct).)*?)\} " + list(pairs)[out.index(got) - 1] + ";", open(header).read(), flags=re.S).group(1)
        assert len(re.findall(r"[,;]", re.sub(r"/\*.*?\*/", "", body, flags=re.S))) == len(cls._fields_)


def test_python_entry_points_refuse_without_a_gpu():
    u8 = dict(dtype=torch.uint8)
    with pytest.raises(_lib.MoondreamHipError, match="GPU"):
        BlockCache(2, 40, 2, 64, device="cpu")
    good = [torch.zeros(2, 2, 64, 64, **u8), torch.zeros(2, 2, 64, 64, **u8), torch.zeros(2, 2, 2, **u8), torch.zeros(2, 2, 2, **u8)]
    with pytest.raises(_lib.MoondreamHipError, match="GPU"):
        BlockCache.of(*good)
    for i, bad in ((0, torch.zeros(2, 2, 64, 72, **u8)), (0, torch.zeros(2, 2, 33, 64, **u8)), (1, torch.zeros(2, 2, 32, 64, **u8)), (2, torch.zeros(2, 2, 4, **u8)),
                   (3, torch.zeros(2, 2, 2)), (0, torch.zeros(2, 2, 64, 128, **u8)[..., :64]), (0, torch.zeros(4, 2, 64, 64, **u8)[::2])):
        with pytest.raises(ValueError):
            BlockCache.of(*[bad if j == i else t for j, t in enumerate(good)])
    with pytest.raises(ValueError):
        BlockCache(0, 32, 1, 64, device="cpu")
    x, s = torch.zeros(4, 10), torch.zeros(2, 2)
    with pytest.raises(_lib.MoondreamHipError, match="GPU"):
        select_beams(x, s)
    for bad in (dict(logits=x[:3]), dict(logits=x.double()), dict(scores=torch.zeros(4, 1)), dict(logits=torch.zeros(34, 10), scores=torch.zeros(2, 17)), dict(end_id=10),
                dict(ended=torch.zeros(2, 2, dtype=torch.int32)), dict(logits=torch.zeros(4, 20)[:, ::2]), dict(logits=torch.zeros(1, 10).expand(4, 10)),
                dict(logits=torch.zeros(4, 0))):
        with pytest.raises(ValueError):
            select_beams(**{**dict(logits=x, scores=s), **bad})
    p, st = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(4, 8)
    with pytest.raises(_lib.MoondreamHipError, match="GPU"):
        reorder_states([st], p)
    reorder_states([], p)
    reorder_states([st[:, :0]], p)
    for args, kw in ((([st[:3]], p), {}), (([st], p[0]), {}), (([st], torch.zeros(1, 17, dtype=torch.int32)), {}), (([st], p), dict(into=[])), (([st], p), dict(into=[st.double()])),
                     (([st], p), dict(into=[torch.zeros(4, 16)[:, ::2]])), (([st], p), dict(slot_dim=1, into=[st])), (([st], p), dict(slot_dim=2)),
                     (([torch.zeros(4, 6, 6, 6, 6)[:, ::2, ::2, ::2, ::2]], p), {})):
        if kw.get("slot_dim") == 1:
            kw = dict(slot_dim=1, into=[torch.zeros(4, 4)])
        with pytest.raises(ValueError):
            reorder_states(*args, **kw)


def test_runs_of_views():
    def runs(t, slot_dim):
        return _runs(tuple(t.shape), t.stride(), t.element_size(), slot_dim, "x")

    slab = torch.zeros(6, 4, 3, 40, 8)
    assert runs(slab, 1) == (3 * 40 * 8 * 4, (1, 0), (6, 4 * 3 * 40 * 8 * 4), 3 * 40 * 8 * 4)
    assert runs(slab[:, :, :, 5:9], 1) == (3 * 40 * 8 * 4, (6, 4 * 3 * 40 * 8 * 4), (3, 40 * 8 * 4), 4 * 8 * 4)
    assert runs(slab[0], 0) == (3 * 40 * 8 * 4, (1, 0), (1, 0), 3 * 40 * 8 * 4)
    assert runs(torch.zeros(4, dtype=torch.uint8), 0) == (1, (1, 0), (1, 0), 1)


def test_the_oracle_rounds_as_torch_does():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(4000, generator=g) * 100, torch.randn(4000, generator=g) * 0.01, torch.arange(-448, 449).float() / 7])
    x = x.clamp(-448, 448)
    codes = x.to(torch.float8_e4m3fn)
    assert torch.equal(U.e4m3(x), codes.double()) and torch.equal(U.value_of(codes.view(torch.uint8)), codes.double())
    for top, e in ((448.0, 0), (448.5, 1), (449.0, 1), (224.0, -1), (896.0, 1), (897.0, 2), (1e-30, U.LOW), (1e30, U.HIGH), (0.0, U.LOW)):
        assert U.exponent(top) == e
