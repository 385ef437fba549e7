"""Attention over a quantised, paged key-value cache, on torch tensors: the operators that a language model's server runs for
each step's new or drafted tokens.

    cache = KvCache.allocate(pages, kv_heads, page_tokens, head_dim, codes=torch.int8)
    q = qkv_to_cache(cache, q, k, v, slots, q_weight, k_weight, cos, sin, positions)       # norm, rotate, quantise, store
    o = tree_attention(q, cache, page_table, context, q_start, max_new=..., max_context=..., mask=...)

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


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, pairs: bool = False, q_out=None, k_out=None):
    """RMS norm of every head of q [tokens, q_heads, head_dim] and k [tokens, kv_heads, head_dim] and rotation by position.

    Weights None: no norm; cos and sin None: no rotation. cos and sin are [positions, rotated / 2]; elements i and
    i + rotated / 2 turn together, or 2i and 2i + 1 with pairs. q_out and k_out may be q and k. Returns (q_out, k_out)."""
    return _native.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, pairs, q_out, k_out)


def qkv_to_cache(cache: KvCache, q, k, v, slots, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, pairs: bool = False, q_out=None):
    """qk_norm_rope, with the keys and values [tokens, kv_heads, head_dim] quantised into the cache's slots (int32; one
    outside of the cache stores nothing) in the same launch. Returns q_out."""
    return _native.qkv_to_cache(q, k, q_weight, k_weight, cos, sin, positions, eps, pairs, v, slots, cache._tensors, q_out)


def kv_write(cache: KvCache, k, v, slots) -> None:
    """Quantises keys and values [tokens, kv_heads, head_dim] into the cache's slots."""
    _native.kv_write(cache._tensors, k, v, slots)


def kv_read(cache: KvCache, slots, *, dtype=_torch.bfloat16, k_out=None, v_out=None):
    """The cache's slots as (keys, values) [len(slots), kv_heads, head_dim]."""
    if dtype not in _HALVES:
        raise ValueError("dtype has to be torch.bfloat16 or torch.float16")
    return _native.kv_read(cache._tensors, slots, _HALVES[dtype], k_out, v_out)


def tree_attention(q, cache: KvCache, page_table, context, q_start, *, max_new: int, max_context: int, mask=None, scale: float | None = None, out=None, lse=None):
    """Attention of new tokens' queries q [tokens, q_heads, head_dim] over the cache.

    Sequence b has context[b] (at most max_context) tokens in the cache and behind them its new ones, rows q_start[b] to
    q_start[b + 1] (at most max_new) of q; its token j is in page page_table[b, j // page_tokens]. Bit u % 64 of
    mask[row, u // 64] (int64) says that a row sees new token u; without a mask new token t sees the new tokens 0 to t.
    All of them see the whole context. Rows that see nothing are zero, and so are those of no sequence (a padded batch's).
    lse [tokens, q_heads] float32 receives the logarithm of the sum of exponentials if it is given. Returns out."""
    return _native.tree_attention(q, cache._tensors, page_table, context, q_start, max_new, max_context, mask, scale, out, lse)
