"""Attention over a quantised, paged key-value cache, on torch tensors: the operators that a language model's server runs for
each step's new or drafted tokens.

    cache = KvCache.allocate(pages, kv_heads, page_tokens, head_dim, codes=torch.int8)
    q = qkv_to_cache(cache, q, k, v, slots, q_weight, k_weight, cos, sin, positions)       # norm, rotate, quantise, store
    o = tree_attention(q, cache, page_table, context, q_start, max_new=..., max_context=..., mask=...)

Thin bindings of the C ABI (include/fklhip.h has the definitions of the operators and the cache's layout): tensors are passed
on by address, the work runs on torch's current stream, and what does not fit raises before anything is launched.  Outputs
are allocated by torch unless they are given.  There is no other path: without libfklhip.so, or on CPU tensors, calls raise.

The library the C ABI answers to has these operators as FK/algorithms/attention/ (attention, split decoding, int8 and fp8
cache reads).
"""
from __future__ import annotations

import ctypes as _C
import struct as _struct

import torch as _torch

from . import check as _check, lib as _lib

_TYPES = {_torch.bfloat16: 0, _torch.float16: 1}
_CODES = {_torch.int8: 0, _torch.float8_e4m3fn: 1}

# struct fklhip_kv_cache, fklhip_rows, fklhip_heads, fklhip_attention of include/fklhip.h
_CACHE = _struct.Struct("@4Pq4i")
_ROWS = _struct.Struct("@Pqq")
_HEADS = _struct.Struct("@" + "Pqq" * 5 + "6Pqq6if4x")
_ATTENTION = _struct.Struct("@" + "Pqq" * 2 + "6PQqq6if4x")

_lib_calls = None


def _calls():
    global _lib_calls
    if _lib_calls is None:
        l = _lib()
        p, c = _C.c_void_p, _C.c_char_p            # structures go as their bytes
        l.fklhip_qk_norm_rope.argtypes = [c, p]
        l.fklhip_qkv_to_cache.argtypes = [c, c, p]
        l.fklhip_kv_write.argtypes = [c, c, c, p, _C.c_int64, _C.c_int, p]
        l.fklhip_kv_read.argtypes = [c, p, _C.c_int64, c, c, _C.c_int, p]
        l.fklhip_tree_attention.argtypes = [c, c, p]
        l.fklhip_tree_attention_workspace.argtypes = [c, c, _C.POINTER(_C.c_uint64)]
        l.fklhip_argument_error.argtypes = [_C.POINTER(c)]
        _lib_calls = l
    return _lib_calls


def _raise(code: int, what: str) -> None:
    if code == 10003:
        text = _C.c_char_p()
        _calls().fklhip_argument_error(_C.byref(text))
        raise ValueError(f"{what}: {text.value.decode()}")
    _check(code, what)


def _stream(t) -> int:
    """torch's current stream of the tensor's device, which has to be the current one (a kernel is launched on that)."""
    index = t.device.index
    if index != _torch._C._cuda_getDevice():
        raise ValueError(f"{t.device} is not the current device")
    return _torch._C._cuda_getCurrentRawStream(index)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(x, name: str, tokens: int, heads: int, dim: int, dtype, device):
    """(address, token stride, head stride) of rows [tokens, heads, dim]."""
    if x.shape != (tokens, heads, dim) or x.dtype != dtype or x.device != device or (x.stride(2) != 1 and dim != 1):
        raise ValueError(f"{name} has to be [{tokens}, {heads}, {dim}] of {dtype} on {device} with a tight last dimension, not {tuple(x.shape)} of {x.dtype} on {x.device}")
    s = x.stride()
    return x.data_ptr(), s[0], s[1]


def _ints(x, name: str, shape, device) -> int:
    if x.dtype != _torch.int32 or tuple(x.shape) != tuple(shape) or x.device != device or not x.is_contiguous():
        raise ValueError(f"{name} has to be {list(shape)} of torch.int32 on {device}, contiguous")
    return x.data_ptr()




class KvCache:
    """A paged cache of keys and values in 8 bits with a float32 scale per token and head.

    k        [pages, kv_heads, page_tokens, head_dim]          int8 or float8_e4m3fn
    v        [pages, kv_heads, page_tokens / 4, head_dim, 4]   four consecutive tokens of one element side by side
    k_scale  [pages, kv_heads, page_tokens] float32, v_scale the same
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page_tokens", "head_dim", "device", "_bytes")

    def __init__(self, k, v, k_scale, v_scale):
        shape = k.shape
        _need(k.dim() == 4 and k.dtype in _CODES, "k has to be [pages, kv_heads, page_tokens, head_dim] of torch.int8 or torch.float8_e4m3fn")
        pages, heads, page, dim = shape
        _need(v.shape == (pages, heads, page // 4, dim, 4) and v.dtype == k.dtype, f"v has to be [{pages}, {heads}, {page // 4}, {dim}, 4] of {k.dtype}")
        _need(k_scale.shape == shape[:3] and v_scale.shape == shape[:3] and k_scale.dtype == _torch.float32 and v_scale.dtype == _torch.float32,
              f"k_scale and v_scale have to be [{pages}, {heads}, {page}] of torch.float32")
        device = k.device
        _need(device.type == "cuda" and v.device == device and k_scale.device == device and v_scale.device == device, "a cache is on one GPU")
        _need(k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous(), "a cache's tensors have to be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_tokens, self.head_dim, self.device = pages, heads, page, dim, device
        self._bytes = _CACHE.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, page, dim, _CODES[k.dtype])

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_tokens: int, head_dim: int, codes=_torch.int8, device="cuda"):
        """An empty cache (its contents are whatever the memory held: attention reads no token that was not written)."""
        _need(codes in _CODES, "codes have to be torch.int8 or torch.float8_e4m3fn")
        k = _torch.empty((pages, kv_heads, page_tokens, head_dim), dtype=codes, device=device)
        v = _torch.empty((pages, kv_heads, page_tokens // 4, head_dim, 4), dtype=codes, device=device)
        scales = [_torch.empty((pages, kv_heads, page_tokens), dtype=_torch.float32, device=device) for _ in range(2)]
        return cls(k, v, *scales)


def _heads(q, k, v, q_weight, k_weight, cos, sin, positions, slots, eps, pairs, q_out, k_out):
    _need(q.dim() == 3 and k.dim() == 3, "q and k have to be [tokens, heads, head_dim]")
    (tokens, q_heads, dim), kv_heads = q.shape, k.shape[1]
    dtype, device = q.dtype, q.device
    _need(dtype in _TYPES, "rows have to be torch.bfloat16 or torch.float16")
    _need(device.type == "cuda", "rows have to be on a GPU")
    _need((q_weight is None) == (k_weight is None), "weights for both of q and k, or for none")
    _need((cos is None) == (sin is None), "cos and sin, or neither")
    none = (0, 0, 0)
    weights = (0, 0)
    if q_weight is not None:
        for w in (q_weight, k_weight):
            _need(w.shape == (dim,) and w.dtype == dtype and w.device == device and w.is_contiguous(), f"weights have to be [{dim}] of {dtype} on {device}, contiguous")
        weights = q_weight.data_ptr(), k_weight.data_ptr()
    tables, rows, half = (0, 0, 0), 0, 0
    if cos is not None:
        rows, half = cos.shape
        _need(sin.shape == (rows, half) and cos.dtype == sin.dtype == _torch.float32 and cos.device == sin.device == device and cos.is_contiguous() and sin.is_contiguous(),
              f"cos and sin have to be [positions, rotated / 2] of torch.float32 on {device}, contiguous")
        tables = cos.data_ptr(), sin.data_ptr(), _ints(positions, "positions", (tokens,), device)
    return _HEADS.pack(
        *_rows(q, "q", tokens, q_heads, dim, dtype, device), *_rows(k, "k", tokens, kv_heads, dim, dtype, device),
        *(none if v is None else _rows(v, "v", tokens, kv_heads, dim, dtype, device)),
        *_rows(q_out, "q_out", tokens, q_heads, dim, dtype, device), *(none if k_out is None else _rows(k_out, "k_out", tokens, kv_heads, dim, dtype, device)),
        *weights, *tables, 0 if slots is None else _ints(slots, "slots", (tokens,), device),
        tokens, rows, q_heads, kv_heads, dim, 2 * half, 1 if pairs else 0, _TYPES[dtype], eps)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, pairs: bool = False, q_out=None, k_out=None):
    """RMS norm of every head of q [tokens, q_heads, head_dim] and k [tokens, kv_heads, head_dim] and rotation by position.

    Weights None: no norm; cos and sin None: no rotation. cos and sin are [positions, rotated / 2]; elements i and
    i + rotated / 2 turn together, or 2i and 2i + 1 with pairs. q_out and k_out may be q and k. Returns (q_out, k_out)."""
    if q_out is None:
        q_out = _torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k_out is None:
        k_out = _torch.empty(k.shape, dtype=k.dtype, device=k.device)
    args = _heads(q, k, None, q_weight, k_weight, cos, sin, positions, None, eps, pairs, q_out, k_out)
    code = _calls().fklhip_qk_norm_rope(args, _stream(q))
    if code:
        _raise(code, "qk_norm_rope")
    return q_out, k_out


def qkv_to_cache(cache: KvCache, q, k, v, slots, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, pairs: bool = False, q_out=None):
    """qk_norm_rope, with the keys and values [tokens, kv_heads, head_dim] quantised into the cache's slots (int32; one
    outside of the cache stores nothing) in the same launch. Returns q_out."""
    if q_out is None:
        q_out = _torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _need(v is not None and slots is not None, "v and slots are needed")
    _need(cache.device == q.device, "the cache is on another device")
    args = _heads(q, k, v, q_weight, k_weight, cos, sin, positions, slots, eps, pairs, q_out, None)
    code = _calls().fklhip_qkv_to_cache(args, cache._bytes, _stream(q))
    if code:
        _raise(code, "qkv_to_cache")
    return q_out


def kv_write(cache: KvCache, k, v, slots) -> None:
    """Quantises keys and values [tokens, kv_heads, head_dim] into the cache's slots."""
    tokens = k.shape[0]
    _need(k.dtype in _TYPES, "rows have to be torch.bfloat16 or torch.float16")
    k_rows = _ROWS.pack(*_rows(k, "k", tokens, cache.kv_heads, cache.head_dim, k.dtype, cache.device))
    v_rows = _ROWS.pack(*_rows(v, "v", tokens, cache.kv_heads, cache.head_dim, k.dtype, cache.device))
    code = _calls().fklhip_kv_write(cache._bytes, k_rows, v_rows, _ints(slots, "slots", (tokens,), cache.device), tokens, _TYPES[k.dtype], _stream(k))
    if code:
        _raise(code, "kv_write")


def kv_read(cache: KvCache, slots, *, dtype=_torch.bfloat16, k_out=None, v_out=None):
    """The cache's slots as (keys, values) [len(slots), kv_heads, head_dim]."""
    _need(dtype in _TYPES, "dtype has to be torch.bfloat16 or torch.float16")
    _need(slots.dim() == 1, "slots has to have one dimension")
    tokens = slots.shape[0]
    shape = (tokens, cache.kv_heads, cache.head_dim)
    if k_out is None:
        k_out = _torch.empty(shape, dtype=dtype, device=cache.device)
    if v_out is None:
        v_out = _torch.empty(shape, dtype=dtype, device=cache.device)
    k_rows, v_rows = (_ROWS.pack(*_rows(x, name, *shape, dtype, cache.device)) for x, name in ((k_out, "k_out"), (v_out, "v_out")))
    code = _calls().fklhip_kv_read(cache._bytes, _ints(slots, "slots", (tokens,), cache.device), tokens, k_rows, v_rows, _TYPES[dtype], _stream(k_out))
    if code:
        _raise(code, "kv_read")
    return k_out, v_out


def tree_attention(q, cache: KvCache, page_table, context, q_start, *, max_new: int, max_context: int, mask=None, scale: float | None = None, out=None, lse=None):
    """Attention of new tokens' queries q [tokens, q_heads, head_dim] over the cache.

    Sequence b has context[b] (at most max_context) tokens in the cache and behind them its new ones, rows q_start[b] to
    q_start[b + 1] (at most max_new) of q; its token j is in page page_table[b, j // page_tokens]. Bit u % 64 of
    mask[row, u // 64] (int64) says that a row sees new token u; without a mask new token t sees the new tokens 0 to t.
    All of them see the whole context. Rows that see nothing are zero. lse [tokens, q_heads] float32 receives the logarithm
    of the sum of exponentials if it is given. Returns out."""
    _need(q.dim() == 3 and q.dtype in _TYPES and q.device == cache.device, "q has to be [tokens, q_heads, head_dim] of torch.bfloat16 or torch.float16 on the cache's device")
    tokens, q_heads, dim = q.shape
    _need(dim == cache.head_dim, "q and the cache have heads of different sizes")
    device = cache.device
    if out is None:
        out = _torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device)
    batch, entries = page_table.shape
    mask_ptr = words = 0
    if mask is not None:
        _need(mask.dim() == 2 and mask.shape[0] == tokens and mask.dtype == _torch.int64 and mask.device == device and mask.is_contiguous(), f"mask has to be [{tokens}, words] of torch.int64 on {device}, contiguous")
        mask_ptr, words = mask.data_ptr(), mask.shape[1]
    lse_ptr = 0
    if lse is not None:
        _need(lse.shape == (tokens, q_heads) and lse.dtype == _torch.float32 and lse.device == device and lse.is_contiguous(), f"lse has to be [{tokens}, {q_heads}] of torch.float32 on {device}, contiguous")
        lse_ptr = lse.data_ptr()
    fields = [*_rows(q, "q", tokens, q_heads, dim, q.dtype, device), *_rows(out, "out", tokens, q_heads, dim, q.dtype, device), lse_ptr,
              _ints(page_table, "page_table", (batch, entries), device), _ints(context, "context", (batch,), device), _ints(q_start, "q_start", (batch + 1,), device), mask_ptr,
              0, 0, tokens, entries, batch, max_new, max_context, words, q_heads, _TYPES[q.dtype], dim ** -0.5 if scale is None else scale]
    calls = _calls()
    args = _ATTENTION.pack(*fields)
    needed = _C.c_uint64()
    code = calls.fklhip_tree_attention_workspace(args, cache._bytes, _C.byref(needed))
    if code:
        _raise(code, "tree_attention")
    if needed.value:
        # torch's allocator gives the memory back to this stream when the work that uses it has been enqueued
        workspace = _torch.empty(needed.value, dtype=_torch.uint8, device=device)
        fields[11:13] = workspace.data_ptr(), needed.value
        args = _ATTENTION.pack(*fields)
    code = calls.fklhip_tree_attention(args, cache._bytes, _stream(q))
    if code:
        _raise(code, "tree_attention")
    return out
