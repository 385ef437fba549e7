"""What the operators of a step around attention refuse, without a GPU: the C ABI's checks (nothing is launched, pointers are not
followed) and the Python bindings'."""
import ctypes as C
import os
import re

import pytest
import torch

import fusedkernellibrary_amd as fkl
from fusedkernellibrary_amd import attention as ops
from test_attention_refusals import AT, I32, I64, P, Cache, a_cache, an_attention, refused, some_heads, some_rows


class Tables(C.Structure):
    _fields_ = [(n, P) for n in ("page_table", "held", "context", "fresh", "free_pages", "available", "parents", "q_start", "slots", "positions", "held_out", "left", "mask")] + [
        (n, I64) for n in ("tokens", "page_table_stride", "free_count")] + [(n, I32) for n in ("batch", "page_tokens", "max_new", "mask_words")]


def some_tables(**more):
    return Tables(**{**dict(page_table=AT, held=AT, context=AT, fresh=AT, free_pages=AT, available=AT, q_start=AT, slots=AT, positions=AT, held_out=2 * AT, left=2 * AT, tokens=4, page_table_stride=3,
                            free_count=5, batch=2, page_tokens=16, max_new=2), **more})


class Drafts(C.Structure):
    _fields_ = [(n, P) for n in ("target", "draft", "ids", "q_start", "parents", "uniforms", "path", "count", "out", "workspace")] + [("workspace_bytes", C.c_uint64)] + [
        (n, I64) for n in ("tokens", "target_stride", "draft_stride")] + [(n, I32) for n in ("batch", "max_new", "vocab", "type")]


def some_drafts(**more):
    return Drafts(**{**dict(target=AT, ids=AT, q_start=AT, uniforms=AT, path=AT, count=AT, out=AT, workspace=AT, workspace_bytes=1 << 30, tokens=6, target_stride=100, draft_stride=100, batch=2,
                            max_new=3, vocab=100, type=2), **more})


class Axes(C.Structure):
    _fields_ = [("stride", I64), ("count", I32), ("of_pair", C.c_uint8 * 128)]


class Scores(C.Structure):
    _fields_ = [(n, P) for n in ("slopes", "positions", "first", "prefix")] + [("cap", C.c_float)]


STRUCTURES = [("fklhip_scores", Scores, 40), ("fklhip_tables", Tables, 144), ("fklhip_drafts", Drafts, 128), ("fklhip_axes", Axes, 144)]


@pytest.mark.parametrize("name,mirror,size", STRUCTURES)
def test_structures_are_the_headers(name, mirror, size):
    """Field for field, in order, and of the sizes that C gives them."""
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fklhip.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, re.S)[1], flags=re.S)
    fields = [re.sub(r"\[.*?\]|[^\w]", "", part.split()[-1]) for line in body.split(";") if line.strip() for part in line.split(",")]
    assert fields == [f[0] for f in mirror._fields_] and C.sizeof(mirror) == size


@pytest.mark.parametrize("change,word", [
    (dict(page_tokens=48), "page_tokens"), (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=512), "page_tokens"), (dict(tokens=-1), "negative"), (dict(tokens=1 << 30), "2^30"),
    (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(max_new=-1), "max_new"), (dict(max_new=1 << 30), "max_new"), (dict(page_table_stride=-1), "page table"),
    (dict(page_table_stride=1 << 30), "page table"), (dict(page_table_stride=1 << 27), "2^30"), (dict(free_count=-1), "free_count"), (dict(free_count=1 << 31), "free_count"),
    (dict(parents=AT, mask=AT), "mask_words"), (dict(parents=AT, mask=AT, mask_words=1, max_new=65), "mask_words"), (dict(parents=AT, mask_words=1), "mask"), (dict(q_start=None), "q_start"),
    (dict(available=None), "available"), (dict(left=None), "left"), (dict(held=None), "lengths"), (dict(held_out=None), "lengths"), (dict(page_table=None), "page_table"),
    (dict(free_pages=None), "free_pages"), (dict(slots=None), "slots"), (dict(positions=None), "positions"), (dict(context=AT + 2), "aligned"), (dict(parents=AT, mask=AT + 4, mask_words=1), "aligned"),
    (dict(held_out=AT), "other arrays"), (dict(left=AT), "other arrays")])
def test_tables(change, word):
    refused(fkl.lib().fklhip_step_tables(C.byref(some_tables(**change)), None), word)
    refused(fkl.lib().fklhip_step_tables(None, None), "no tables")


def test_bindings_of_tables():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.step_tables(i.view(2, 2), i[:2], i[:2], i[:2], i, i[:1], page_tokens=16, tokens=2, max_new=1)
    with pytest.raises(ValueError, match="page_table"):
        ops.step_tables(i, i, i, i, i, i[:1], page_tokens=16, tokens=2, max_new=1)
    with pytest.raises(ValueError, match="tensor"):
        ops.step_tables([1], i, i, i, i, i[:1], page_tokens=16, tokens=2, max_new=1)


@pytest.mark.parametrize("change,word", [
    (dict(type=3), "type"), (dict(type=-1), "type"), (dict(tokens=-1), "negative"), (dict(tokens=1 << 30), "2^30"), (dict(batch=-1), "batch"), (dict(batch=65536), "batch"),
    (dict(max_new=-1), "max_new"), (dict(max_new=1025), "max_new"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1), "vocab"), (dict(q_start=None), "q_start"), (dict(path=None), "results"),
    (dict(count=None), "results"), (dict(out=None), "results"), (dict(target=None), "target"), (dict(ids=None), "ids"), (dict(uniforms=None), "uniforms"), (dict(draft=AT, parents=AT), "chains"),
    (dict(target=AT + 2), "aligned"), (dict(type=0, target=AT + 1), "aligned"), (dict(draft=AT + 2), "aligned"), (dict(parents=AT + 1), "aligned"), (dict(out=AT + 2), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=2 * 8 + 2 * 11 * 4 - 1), "workspace"), (dict(workspace=AT + 4), "8 bytes")])
def test_drafts(change, word):
    refused(fkl.lib().fklhip_verify_drafts(C.byref(some_drafts(**change)), None), word)
    refused(fkl.lib().fklhip_verify_drafts(None, None), "no drafts")


def test_workspaces_of_drafts():
    l, need = fkl.lib(), C.c_uint64()
    of = lambda **c: (l.fklhip_verify_drafts_workspace(C.byref(some_drafts(**c)), C.byref(need)), need.value)      # noqa: E731
    assert of() == (0, 2 * 8 + 2 * 11 * 4) and of(vocab=4097) == (0, 4 * 8 + 2 * 11 * 4) and of(batch=0) == (0, 0) and of(max_new=0) == (0, 0)
    refused(l.fklhip_verify_drafts_workspace(C.byref(some_drafts()), None), "answer")
    refused(l.fklhip_verify_drafts_workspace(C.byref(some_drafts(vocab=0)), C.byref(need)), "vocab")
    for nothing in (dict(batch=0, workspace=None), dict(max_new=0, workspace=None)):
        assert l.fklhip_verify_drafts(C.byref(some_drafts(**nothing)), None) == 0


def keep(caches=2, stride=3, table=AT, context=AT, path=AT, count=AT, batch=2, most=3, **more):
    l = fkl.lib()
    l.fklhip_kv_keep.argtypes = [P, I32, P, I64, P, P, P, I32, I32, P]
    these = (Cache * max(1, caches))(*[a_cache(**{n: (i + 1) * AT for n in ("k", "v", "k_scale", "v_scale")}) for i in range(max(0, min(caches, 1025)))])
    for name, value in more.items():
        setattr(these[1], name, value)
    return l.fklhip_kv_keep(these, caches, table, stride, context, path, count, batch, most, None)


@pytest.mark.parametrize("change,word", [
    (dict(caches=-1), "layers"), (dict(caches=1025), "layers"), (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(most=-1), "max_new"), (dict(most=(1 << 20) + 1), "max_new"),
    (dict(stride=-1), "page_table_stride"), (dict(stride=1 << 31), "page_table_stride"), (dict(k=AT), "twice"), (dict(v=AT), "twice"), (dict(k_scale=AT), "twice"), (dict(v_scale=AT), "twice"),
    (dict(pages=9), "different sizes"), (dict(kv_heads=3), "different sizes"), (dict(page_tokens=32), "different sizes"), (dict(head_dim=128), "different sizes"), (dict(codes=1), "different sizes"),
    (dict(codes=5), "codes"), (dict(table=None), "page_table"), (dict(context=None), "context"), (dict(path=None), "path"), (dict(count=None), "count"), (dict(path=AT + 2), "aligned")])
def test_keep(change, word):
    refused(keep(**change), word)


def test_keeping_nothing():
    for nothing in (dict(caches=0), dict(batch=0), dict(most=0), dict(stride=0)):
        assert keep(**nothing) == 0


def test_bindings_of_drafts_and_kept_rows():
    x, i = torch.zeros((2, 9)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.verify_drafts(x, i, i, x[:, 0], max_new=2)
    with pytest.raises(ValueError, match="float32, torch.bfloat16"):
        ops.verify_drafts(x.double(), i, i, x[:, 0], max_new=2)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.verify_drafts(x[0], i, i, x[:, 0], max_new=2)
    with pytest.raises(ValueError, match="q_start"):
        ops.verify_drafts(x, i, i[:0], x[:, 0], max_new=2)
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_keep([], i.view(2, 1), i, i.view(2, 1), i)


def some_axes(count=3, of_pair=(0, 1, 2)):
    return Axes(3, count, (C.c_uint8 * 128)(*of_pair))


@pytest.mark.parametrize("axes,word", [(some_axes(0), "1 to 4"), (some_axes(5), "1 to 4"), (some_axes(2), "none of them"), (some_axes(4, (0,) * 31 + (4,)), "none of them"), (None, "no axes")])
def test_axes(axes, word):
    refused(fkl.lib().fklhip_qk_norm_rope_axes(C.byref(some_heads()), C.byref(axes) if axes else None, None), word)
    refused(fkl.lib().fklhip_qkv_to_cache_axes(C.byref(some_heads()), C.byref(axes) if axes else None, C.byref(a_cache()), None), word)


def test_axes_of_pairs_that_do_not_turn_are_not_looked_at():
    assert fkl.lib().fklhip_qk_norm_rope_axes(C.byref(some_heads(tokens=0)), C.byref(some_axes(4, (0,) * 32 + (9,))), None) == 0
    refused(fkl.lib().fklhip_qkv_to_cache_axes(C.byref(some_heads()), C.byref(some_axes()), None, None), "no cache")


@pytest.mark.parametrize("change,call,word", [
    (dict(cap=-1.0), {}, "cap"), (dict(cap=2.0 ** -7), {}, "cap"), (dict(cap=513.0), {}, "cap"), (dict(cap=float("nan")), {}, "cap"), (dict(cap=float("inf")), {}, "cap"),
    (dict(slopes=AT + 2), {}, "aligned"), (dict(positions=AT + 1), {}, "aligned"), (dict(first=AT + 2), {}, "aligned"), (dict(prefix=AT + 2), {}, "aligned"),
    (dict(prefix=AT), dict(mask=AT, mask_words=1), "prefix and a mask"), (dict(cap=4.0), dict(type=3), "type"), (dict(cap=4.0), dict(q=some_rows(data=AT + 2)), "16 bytes"),
    (dict(first=AT), dict(max_context=1 << 20, page_table_stride=1 << 18), "workspace")])
def test_scores(change, call, word):
    refused(fkl.lib().fklhip_shaped_attention(C.byref(an_attention(**call)), C.byref(Scores(**change)), C.byref(a_cache()), None), word)


def test_shaping_nothing():
    l = fkl.lib()
    refused(l.fklhip_shaped_attention(C.byref(an_attention()), None, C.byref(a_cache()), None), "no scores")
    for nothing in (dict(tokens=0), dict(batch=0), dict(max_new=0)):
        assert l.fklhip_shaped_attention(C.byref(an_attention(**nothing)), C.byref(Scores(cap=3.0)), C.byref(a_cache()), None) == 0
