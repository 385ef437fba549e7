"""Outputs of the attention operators whose rows share memory are refused, without a GPU (every call here is refused: at its output, or at
what is looked at after it)."""
import ctypes as C
import random

import pytest

import fusedkernellibrary_amd as fkl
from test_attention_refusals import AT, P, I64, Rows, a_cache, an_attention, refused, some_heads, some_rows, text

DIM = 64


def attend(tokens, heads, token_stride, head_stride):
    """What a call with such an output is refused for: its output, or the lengths that are missing."""
    rows = Rows(AT, heads * DIM, DIM)
    call = an_attention(q=rows, out=Rows(AT, token_stride, head_stride), tokens=tokens, q_heads=heads, context=None)
    assert fkl.lib().fklhip_tree_attention(C.byref(call), C.byref(a_cache(kv_heads=1)), None) == 10003
    return text()


def overlap(tokens, heads, token_stride, head_stride):
    seen = set()
    for t in range(tokens):
        for h in range(heads):
            row = set(range(t * token_stride + h * head_stride, t * token_stride + h * head_stride + DIM, 8))
            if seen & row:
                return True
            seen |= row
    return False


@pytest.mark.parametrize("seed", range(8))
def test_rows_that_overlap(seed):
    """Strides of all kinds (equal, interleaved, 0, negative) against the rows' places one by one."""
    rng, told = random.Random(seed), [0, 0]
    for _ in range(1500):
        tokens, heads = rng.randint(1, 7), rng.randint(1, 7)
        strides = [rng.choice([0, 8, 56, 64, 72, 128, 64 * heads, 64 * tokens, 64 * heads + 8, 8 * rng.randint(-90, 90)]) for _ in range(2)]
        want = overlap(tokens, heads, *strides)
        got = attend(tokens, heads, *strides)
        assert got == ("rows of an output overlap" if want else "no context or no q_start"), (tokens, heads, strides)
        told[want] += 1
    assert min(told) > 100


def test_strides_beyond_32_bits():
    assert "context" in attend(1 << 20, 4, 1 << 50, 1 << 44) and "overlap" in attend(1 << 20, 4, 1 << 50, 1 << 50) and "context" in attend(1, 1, 0, 0)


def test_every_output():
    l, wide, twice = fkl.lib(), some_rows(2, head_stride=32), some_rows(2, token_stride=0)
    refused(l.fklhip_qk_norm_rope(C.byref(some_heads(q_out=some_rows(head_stride=0))), None), "overlap")
    refused(l.fklhip_qk_norm_rope(C.byref(some_heads(k_out=some_rows(2, token_stride=64))), None), "overlap")
    refused(l.fklhip_qkv_to_cache(C.byref(some_heads(q_out=some_rows(token_stride=0))), C.byref(a_cache()), None), "overlap")
    l.fklhip_kv_read.argtypes = [P, P, I64, P, P, C.c_int, P]
    cache, fine = a_cache(), some_rows(2)
    for k, v in ((wide, fine), (fine, twice)):
        refused(l.fklhip_kv_read(C.addressof(cache), AT, 3, C.addressof(k), C.addressof(v), 0, None), "overlap")
    # inputs may: a row for all tokens, say
    refused(l.fklhip_qk_norm_rope(C.byref(some_heads(q=some_rows(token_stride=0), k=some_rows(2, head_stride=0), q_out=some_rows(head_stride=0))), None), "output")
