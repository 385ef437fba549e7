"""Attention over a quantised, paged key-value cache, on torch tensors: the operators that a language model's server runs for
each step's new or drafted tokens.

    cache = KvCache.allocate(pages, kv_heads, page_tokens, head_dim, codes=torch.int8)
    q = qkv_to_cache(cache, q, k, v, slots, q_weight, k_weight, cos, sin, positions)       # norm, rotate, quantise, store
    o = tree_attention(q, cache, page_table, context, q_start, max_new=..., max_context=..., mask=...)

and around the layers of a step of drafted tokens

    t = step_tables(page_table, held, context, new, free, available, page_tokens=..., tokens=..., max_new=..., parents=...)
    v = verify_drafts(target, tokens, t.q_start, uniforms, max_new=..., parents=...)
    kv_keep(caches, page_table, context, v.path, v.count)

Thin bindings of the C ABI (include/fklhip.h has the definitions of the operators and the cache's layout): tensors are passed
on by address, the work runs on torch's current stream, and what does not fit raises ValueError before anything is launched.
Outputs are allocated by torch unless they are given. The operators serve and do not train: under grad mode an argument that
asks for a gradient is refused, a norm's weights too, and so is a forward-mode tangent. The calls are no operators of torch's
dispatcher, so tracers (torch.jit.trace, make_fx) cannot record them and are refused; a HIP graph can. There is no other path:
without the compiled library, or on CPU tensors, calls raise.

The library the C ABI answers to has these operators as FK/algorithms/attention/ (attention, split decoding, int8 and fp8
cache reads).
"""
from __future__ import annotations

import typing as _typing

import torch as _torch

from . import lib as _lib

_lib()                          # says what is missing if nothing is built
try:
    from . import _attention as _native  # noqa: E402  (csrc/attention/torch_binding.cpp; needs torch and the library loaded)
except ImportError as e:
    raise ImportError("_attention.so is not built, or not for this torch: python -m fusedkernellibrary_amd.build, with a torch for ROCm") from e

_HALVES = {_torch.bfloat16: False, _torch.float16: True}


class KvCache:
    """A paged cache of keys and values in 8 bits with a float32 scale per token and head.

    k        [pages, kv_heads, page_tokens, head_dim]          int8 or float8_e4m3fn
    v        [pages, kv_heads, page_tokens / 4, head_dim, 4]   four consecutive tokens of one element side by side
    k_scale  [pages, kv_heads, page_tokens] float32, v_scale the same

    It is of these tensors for good, and holds nothing of them but the tensors: every call looks at where they are and at what
    they are then. Making one costs next to nothing.
    """

    __slots__ = ("_tensors",)

    def __init__(self, k, v, k_scale, v_scale):
        tensors = k, v, k_scale, v_scale
        _native.check_cache(tensors)
        self._tensors = tensors

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    pages = property(lambda self: self.k.shape[0])
    kv_heads = property(lambda self: self.k.shape[1])
    page_tokens = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])
    codes = property(lambda self: self.k.dtype)
    device = property(lambda self: self.k.device)

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_tokens: int, head_dim: int, codes=_torch.int8, device="cuda"):
        """An empty cache (its contents are whatever the memory held: attention reads no token that was not written)."""
        k = _torch.empty((pages, kv_heads, page_tokens, head_dim), dtype=codes, device=device)
        v = _torch.empty((pages, kv_heads, page_tokens // 4, head_dim, 4), dtype=codes, device=device)
        scales = [_torch.empty((pages, kv_heads, page_tokens), dtype=_torch.float32, device=device) for _ in range(2)]
        return cls(k, v, *scales)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, pairs: bool = False, q_out=None, k_out=None, axes=None):
    """RMS norm of every head of q [tokens, q_heads, head_dim] and k [tokens, kv_heads, head_dim] and rotation by position.

    Weights None: no norm; cos and sin None: no rotation. cos and sin are [positions, rotated / 2]; elements i and
    i + rotated / 2 turn together, or 2i and 2i + 1 with pairs. With axes, a whole number for each of the rotated / 2 pairs,
    positions is [axes, tokens], up to 4, and pair i turns by the positions of axes[i] (an image's or a video's time, height and
    width). q_out and k_out may be q and k. Returns (q_out, k_out)."""
    return _native.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, pairs, q_out, k_out, axes)


def qkv_to_cache(cache: KvCache, q, k, v, slots, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, pairs: bool = False, q_out=None, axes=None):
    """qk_norm_rope, with the keys and values [tokens, kv_heads, head_dim] quantised into the cache's slots (int32; one
    outside of the cache stores nothing) in the same launch. Returns q_out."""
    return _native.qkv_to_cache(q, k, q_weight, k_weight, cos, sin, positions, eps, pairs, v, slots, cache._tensors, q_out, axes)


def kv_write(cache: KvCache, k, v, slots) -> None:
    """Quantises keys and values [tokens, kv_heads, head_dim] into the cache's slots."""
    _native.kv_write(cache._tensors, k, v, slots)


def kv_read(cache: KvCache, slots, *, dtype=_torch.bfloat16, k_out=None, v_out=None):
    """The cache's slots as (keys, values) [len(slots), kv_heads, head_dim]."""
    if dtype not in _HALVES:
        raise ValueError("dtype has to be torch.bfloat16 or torch.float16")
    return _native.kv_read(cache._tensors, slots, _HALVES[dtype], k_out, v_out)


def tree_attention(q, cache: KvCache, page_table, context, q_start, *, max_new: int, max_context: int, mask=None, scale: float | None = None, out=None, lse=None,
                   cap: float | None = None, slopes=None, positions=None, first=None, prefix=None):
    """Attention of new tokens' queries q [tokens, q_heads, head_dim] over the cache.

    Sequence b has context[b] (at most max_context) tokens in the cache and behind them its new ones, rows q_start[b] to
    q_start[b + 1] (at most max_new) of q; its token j is in page page_table[b, j // page_tokens]. Bit u % 64 of
    mask[row, u // 64] (int64) says that a row sees new token u; without a mask new token t sees the new tokens 0 to t.
    All of them see the whole context. Rows that see nothing are zero, and so are those of no sequence (a padded batch's).
    lse [tokens, q_heads] float32 receives the logarithm of the sum of exponentials if it is given. Returns out.

    Scores of another shape: cap (2^-6 to 2^9) makes them cap * tanh(score / cap); slopes [q_heads] float32 takes off slope * (the
    row's position - the key's), which are places in the sequence or, of new tokens, positions [tokens] int32 (step_tables', of
    trees); a key behind its row, as a prefix has them, gains by it, as a bias of slope * (the key's position) has it. Rows that see other keys: none in front of place first[row] (int32; a window, the beginning of the row's document;
    none of a sequence's rows sees what is in front of its first row's, and nothing of that is read), or, without a mask, all in
    front of place prefix[b] (int32) besides those that they see anyway."""
    return _native.tree_attention(q, cache._tensors, page_table, context, q_start, max_new, max_context, mask, scale, out, lse, cap, slopes, positions, first, prefix)


class StepTables(_typing.NamedTuple):
    """What step_tables returns, in one allocation; the names are those of the arguments that take them."""
    q_start: _torch.Tensor          # [batch + 1]
    slots: _torch.Tensor            # [tokens]
    positions: _torch.Tensor        # [tokens]
    held: _torch.Tensor             # [batch]
    available: _torch.Tensor        # [1]
    mask: _torch.Tensor | None      # [tokens, words] int64, of trees


def step_tables(page_table, held, context, new, free, available, *, page_tokens: int, tokens: int, max_new: int, parents=None) -> StepTables:
    """The tables of a step from its requests' lengths, in one launch and without a look at them on the host. All are int32.

    Request b has context[b] tokens in the cache, the first held[b] entries of page_table[b] and new[b] (at most max_new) new
    tokens. The pages that those need are taken from the end of the first `available` [1] entries of free, request by request,
    and written to page_table; held and available are returned as they are afterwards (available is negative by the pages that
    were missing; a token without a page has slot -1). The step has `tokens` rows: rows behind the last request's have slot
    -1, position 0 and an empty mask. With parents [tokens], new token t of a sequence follows its new token
    parents[row] < t (-1: none): its position is context + the number of its ancestors, and its mask has them and itself."""
    return StepTables._make(_native.step_tables(page_table, held, context, new, free, available, page_tokens, tokens, max_new, parents))


class Verified(_typing.NamedTuple):
    """What verify_drafts returns, int32, in one allocation."""
    path: _torch.Tensor             # [batch, max_new]: the accepted rows, counted from the sequence's first; then -1
    count: _torch.Tensor            # [batch]: how many they are
    out: _torch.Tensor              # [batch, max_new]: the tokens that were decided, as many; then -1


def verify_drafts(target, tokens, q_start, uniforms, *, max_new: int, draft=None, parents=None) -> Verified:
    """Drafted tokens against the target's probabilities, by random numbers that are given.

    Sequence b's rows are q_start[b] to q_start[b + 1] (at most max_new, up to 1024): the first is of the last token that is
    decided, the others of drafted ones, tokens[row] (int32). target [tokens, vocabulary] (float32, bfloat16 or float16) has the
    probabilities of what follows each row. Row t follows row parents[row] < t, counted from its sequence's first, or row t - 1.
    The children of the last accepted row are asked in their order: one with token x is accepted if target[parent, x] >
    uniforms[row] * draft[row, x], draft being the probabilities that the tokens were drawn from (of chains), or without draft >
    uniforms[row] * (1 - what the refused children in front of it had). Where none is accepted the next token is drawn from
    max(target - draft, 0) of the refused row, from target without the refused tokens, or from target, by the uniform [0, 1) of
    the sequence's first row. Tokens come out distributed as if drawn from target one by one."""
    return Verified._make(_native.verify_drafts(target, tokens, q_start, uniforms, max_new, draft, parents))


def kv_keep(caches, page_table, context, path, count) -> None:
    """Moves the rows of accepted tokens to where their sequences go on, in a cache or in those of several layers at once: what
    is at place context[b] + path[b, i] of sequence b goes to place context[b] + i, for i from 1 up to count[b]. path (as
    verify_drafts returns it) ascends. No two caches overlap, and no two sequences share a page where something moves."""
    caches = (caches,) if isinstance(caches, KvCache) else caches
    _native.kv_keep(tuple(c._tensors for c in caches), page_table, context, path, count)
