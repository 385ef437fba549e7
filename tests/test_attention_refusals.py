"""What the attention operators refuse, without a GPU: the C ABI's checks (nothing is launched, pointers are not followed) and
the Python bindings'."""
import ctypes as C
import os
import re

import pytest
import torch

import fusedkernellibrary_amd as fkl
from fusedkernellibrary_amd import attention as ops

P, I64, I32 = C.c_void_p, C.c_int64, C.c_int32
EINVAL = 10003


class Cache(C.Structure):
    _fields_ = [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("pages", I64), ("kv_heads", I32), ("page_tokens", I32), ("head_dim", I32), ("codes", I32)]


class Rows(C.Structure):
    _fields_ = [("data", P), ("token_stride", I64), ("head_stride", I64)]


class Heads(C.Structure):
    _fields_ = [(n, Rows) for n in ("q", "k", "v", "q_out", "k_out")] + [(n, P) for n in ("q_weight", "k_weight", "cos", "sin", "positions", "slots")] + [
        ("tokens", I64), ("table_rows", I64)] + [(n, I32) for n in ("q_heads", "kv_heads", "head_dim", "rot_dim", "pairs", "type")] + [("eps", C.c_float)]


class Attention(C.Structure):
    _fields_ = [("q", Rows), ("out", Rows)] + [(n, P) for n in ("lse", "page_table", "context", "q_start", "mask", "workspace")] + [
        ("workspace_bytes", C.c_uint64), ("tokens", I64), ("page_table_stride", I64)] + [(n, I32) for n in ("batch", "max_new", "max_context", "mask_words", "q_heads", "type")] + [
        ("scale", C.c_float)]


AT = 0x1000            # an address that nobody reads


def a_cache(**more):
    return Cache(**{**dict(k=AT, v=AT, k_scale=AT, v_scale=AT, pages=8, kv_heads=2, page_tokens=16, head_dim=64, codes=0), **more})


def some_rows(heads=4, data=AT, token_stride=None, head_stride=64):
    return Rows(data, heads * 64 if token_stride is None else token_stride, head_stride)


def some_heads(**more):
    return Heads(**{**dict(q=some_rows(), k=some_rows(2), v=some_rows(2), q_out=some_rows(), k_out=some_rows(2), cos=AT, sin=AT, positions=AT, slots=AT, tokens=3, table_rows=100,
                           q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, type=0, eps=1e-6), **more})


def an_attention(**more):
    return Attention(**{**dict(q=some_rows(), out=some_rows(), page_table=AT, context=AT, q_start=AT, tokens=3, page_table_stride=4, batch=2, max_new=2, max_context=40, q_heads=4,
                               type=0, scale=0.125), **more})


def text():
    t = C.c_char_p()
    assert fkl.lib().fklhip_argument_error(C.byref(t)) == 0
    return t.value.decode()


def refused(rc, word):
    assert rc == EINVAL and word in text(), (rc, text())


def test_structures_are_the_headers():
    """Field for field, in order, and of the sizes that C gives them."""
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fklhip.h")).read()
    for name, mirror, size in (("fklhip_kv_cache", Cache, 56), ("fklhip_rows", Rows, 24), ("fklhip_heads", Heads, 216), ("fklhip_attention", Attention, 152)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, re.S)[1], flags=re.S)
        fields = [re.sub(r"[^\w]", "", part.split()[-1]) for line in body.split(";") if line.strip() for part in line.split(",")]
        assert fields == [f[0] for f in mirror._fields_] and C.sizeof(mirror) == size


@pytest.mark.parametrize("change,word", [
    (dict(type=2), "type"), (dict(tokens=-1), "negative"), (dict(tokens=1 << 30), "2^30"), (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(rot_dim=72), "rot_dim"),
    (dict(rot_dim=12), "rot_dim"), (dict(q_heads=0), "q_heads"), (dict(kv_heads=70000), "kv_heads"), (dict(pairs=2), "pairs"), (dict(cos=None), "tables"), (dict(positions=None), "positions"),
    (dict(cos=AT + 4), "16 bytes"), (dict(table_rows=0), "tables"), (dict(q_weight=AT), "both"), (dict(q_weight=AT, k_weight=AT + 2), "8 bytes"),
    (dict(q_weight=AT, k_weight=AT, eps=-1.0), "eps"), (dict(positions=AT + 2), "aligned"), (dict(q=Rows(None, 256, 64)), "without data"), (dict(q=some_rows(data=AT + 8)), "16 bytes"),
    (dict(k=some_rows(token_stride=100)), "token stride"), (dict(q_out=some_rows(head_stride=68)), "head stride"), (dict(k_out=Rows(None, 0, 0)), "without data")])
def test_heads(change, word):
    refused(fkl.lib().fklhip_qk_norm_rope(C.byref(some_heads(**change)), None), word)


@pytest.mark.parametrize("change,cache,word", [
    ({}, dict(k=None), "without data"), ({}, dict(v_scale=AT + 4), "16 bytes"), ({}, dict(codes=7), "codes"), ({}, dict(page_tokens=24), "page_tokens"), ({}, dict(page_tokens=512), "page_tokens"),
    ({}, dict(pages=0), "slots"), ({}, dict(pages=1 << 62), "slots"), ({}, dict(kv_heads=3), "other heads"), ({}, dict(head_dim=128), "other heads"), (dict(slots=None), {}, "slots"),
    (dict(v=Rows(None, 0, 0)), {}, "without data"), (dict(slots=AT + 1), {}, "aligned")])
def test_heads_to_a_cache(change, cache, word):
    refused(fkl.lib().fklhip_qkv_to_cache(C.byref(some_heads(**change)), C.byref(a_cache(**cache)), None), word)


def test_write_and_read():
    l, r = fkl.lib(), some_rows(2)
    l.fklhip_kv_write.argtypes = [P, P, P, P, I64, C.c_int, P]
    l.fklhip_kv_read.argtypes = [P, P, I64, P, P, C.c_int, P]
    held = a_cache()
    cache, at = C.addressof(held), C.addressof(r)
    refused(l.fklhip_kv_write(None, at, at, AT, 1, 0, None), "no cache")
    refused(l.fklhip_kv_write(cache, at, at, AT, 1, 5, None), "type")
    refused(l.fklhip_kv_write(cache, at, at, AT, -1, 0, None), "negative")
    refused(l.fklhip_kv_write(cache, at, None, AT, 1, 0, None), "rows")
    refused(l.fklhip_kv_write(cache, at, at, None, 1, 0, None), "slots")
    refused(l.fklhip_kv_read(cache, AT + 2, 1, at, at, 0, None), "aligned")
    odd = some_rows(2, token_stride=130)
    refused(l.fklhip_kv_read(cache, AT, 2, at, C.addressof(odd), 0, None), "token stride")
    assert l.fklhip_kv_write(cache, None, None, None, 0, 0, None) == 0 and l.fklhip_kv_read(cache, None, 0, None, None, 1, None) == 0      # no tokens: nothing to do


@pytest.mark.parametrize("change,cache,word", [
    (dict(type=3), {}, "type"), (dict(tokens=-2), {}, "negative"), ({}, dict(head_dim=72), "64, 96, 128"), (dict(q_heads=5), {}, "multiple of kv_heads"), (dict(batch=65536), {}, "batch"),
    (dict(max_new=-1), {}, "max_new"), (dict(max_context=-1), {}, "max_context"), (dict(max_context=1 << 30), {}, "2^30"), (dict(max_new=1 << 20), {}, "2^20"),
    (dict(tokens=1 << 29, q_heads=8), {}, "query rows"), (dict(page_table_stride=-1), {}, "page_table_stride"), (dict(page_table_stride=1 << 40), {}, "page_table_stride"),
    (dict(scale=float("nan")), {}, "finite"), (dict(scale=float("inf")), {}, "finite"), (dict(q=some_rows(data=AT + 2)), {}, "16 bytes"), (dict(out=some_rows(token_stride=250)), {}, "token stride"),
    (dict(context=None), {}, "context"), (dict(q_start=None), {}, "q_start"), (dict(page_table=None), {}, "page_table"), (dict(mask=AT, mask_words=0), {}, "mask_words"),
    (dict(mask=AT, mask_words=1, max_new=65), {}, "mask_words"), (dict(mask=AT + 4, mask_words=1), {}, "aligned"), (dict(lse=AT + 2), {}, "aligned"),
    (dict(max_context=1 << 20, page_table_stride=1 << 18), {}, "workspace"), ({}, dict(page_tokens=8), "page_tokens")])
def test_attention(change, cache, word):
    refused(fkl.lib().fklhip_tree_attention(C.byref(an_attention(**change)), C.byref(a_cache(**cache)), None), word)


def test_workspaces():
    l = fkl.lib()
    need = C.c_uint64()
    of = lambda **c: (l.fklhip_tree_attention_workspace(C.byref(an_attention(**c)), C.byref(a_cache()), C.byref(need)), need.value)      # noqa: E731
    assert of() == (0, 0)                                                           # short sequences: nobody's work is shared
    rc, some = of(max_context=1 << 20, page_table_stride=1 << 18)
    assert rc == 0 and 0 < some <= 768 * 2 * 16 * 65 * 4
    refused(l.fklhip_tree_attention_workspace(C.byref(an_attention()), C.byref(a_cache()), None), "answer")
    small = an_attention(max_context=1 << 20, page_table_stride=1 << 18, workspace=AT, workspace_bytes=some - 1)
    refused(l.fklhip_tree_attention(C.byref(small), C.byref(a_cache()), None), "smaller")
    askew = an_attention(max_context=1 << 20, page_table_stride=1 << 18, workspace=AT + 4, workspace_bytes=some)
    refused(l.fklhip_tree_attention(C.byref(askew), C.byref(a_cache()), None), "16 bytes")
    for nothing in (dict(tokens=0), dict(batch=0), dict(max_new=0)):
        assert l.fklhip_tree_attention(C.byref(an_attention(**nothing)), C.byref(a_cache()), None) == 0
    assert l.fklhip_argument_error(None) == EINVAL


def test_bindings_refuse_tensors_that_are_not_on_a_gpu():
    k, s = torch.zeros((2, 1, 16, 64), dtype=torch.int8), torch.zeros((2, 1, 16))
    with pytest.raises(ValueError, match="GPU"):
        ops.KvCache(k, k.view(2, 1, 4, 64, 4), s, s)
    with pytest.raises(ValueError, match="int8 or torch.float8_e4m3fn"):
        ops.KvCache(s, s, s, s)
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.qk_norm_rope(x, x, None, None, None, None, None)
    with pytest.raises(ValueError, match="bfloat16 or torch.float16"):
        ops.qk_norm_rope(x.float(), x.float(), None, None, None, None, None)
    with pytest.raises(ValueError, match="tensor"):
        ops.qk_norm_rope(x, 7, None, None, None, None, None)
    with pytest.raises(ValueError, match="for both"):
        ops.qk_norm_rope(x, x, x[0, 0], None, None, None, None)
    with pytest.raises(ValueError, match="arguments"):
        ops._native.tree_attention(1)
