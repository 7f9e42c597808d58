"""A paged K/V cache held in 4 or 8 bits: writing it, reading it back, attending it.

The layout is paged_kv's with elements and their scales in two tensors of bytes
each (QuantizedKV): 32 elements along the head dim share a scale, a power of two
2^(c - 127) in a byte c.  4 bits: e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their
negatives), two to a byte, the even one in the low half; 8 bits: e4m3 (largest
448).  A cache takes 4.25 or 8.25 bits per element where a 16-bit one takes 16:
N(0, 1) rows come back with a relative error (of their norm) of 0.112 in 4 bits
and 0.027 in 8.

A serving step is paged_kv's with this cache in its place; prompts and the tree
half of a verification attend their own 16-bit rows:

    cache = quantized_kv_cache(pages, page_size, Hkv, D, bits=4)
    # prompt: its rows into the pages
    O = prompt_attention(Q, K, V, cu, max_seqlen)
    lens = append_quantized_kv(K, V, cache, table, lens, cu, max_seqlen)
    # verify a draft tree: context and tree, merged; its rows behind the context
    Oc, Lc = prefix_attention_quantized(q, cache, table, lens, cu, max_seqlen)
    Ot, Lt = ragged_attention_with_lse(q, k, v, cu, b, depth, max_seqlen)
    O = fused_lse_merge(...)
    append_quantized_kv(k, v, cache, table, lens, cu, max_seqlen)
    # keep the accepted path; fork a sequence's last page: compact_paged_kv and
    # copy_kv_pages move bytes too, elements and scales one after the other
    new = compact_paged_kv(cache.K, cache.V, table, lens, accepted)
    compact_paged_kv(cache.K_scale, cache.V_scale, table, lens, accepted)

The calls run on torch's current stream, take contexts, offsets and page tables
on the host too and refuse tensors that ask for gradients while autograd records,
as paged_kv's do.
"""
from __future__ import annotations

import math
import operator
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .paged_kv import _lengths, _rows, _table
from .ragged_attn import _SUPPORTED, _device_index, _dtype_code, _launch, _no_grad, _out_like, _rows16

BLOCK = 32  # elements of a scale


class QuantizedKV(NamedTuple):
    """One layer's cache, or the caches of all layers: bytes of elements K, V [...,
    pages, page_size, Hkv, D * bits / 8] and of scales K_scale, V_scale [..., pages,
    page_size, Hkv, D / 32].  K and V are laid out alike (the same strides)."""

    K: torch.Tensor
    V: torch.Tensor
    K_scale: torch.Tensor
    V_scale: torch.Tensor

    def layer(self, i: int) -> "QuantizedKV":
        """Layer i's cache of [layers, ...] tensors (views)."""
        return QuantizedKV(*(t[i] for t in self))


def quantized_kv_cache(
    num_pages: int,
    page_size: int,
    num_kv_heads: int,
    head_dim: int,
    bits: int = 4,
    layers: Optional[int] = None,
    device="cuda",
) -> QuantizedKV:
    """A cache of zeros, with a leading layer dim if layers is given."""
    if bits not in (4, 8):
        raise ValueError(f"bits must be 4 or 8 (got {bits})")
    if head_dim not in (32, 64, 128):
        raise ValueError(f"head_dim {head_dim} not in (32, 64, 128)")
    shape = (num_pages, page_size, num_kv_heads) if layers is None else (layers, num_pages, page_size, num_kv_heads)

    def zeros(n):
        return torch.zeros(*shape, n, dtype=torch.uint8, device=device)

    elements, scales = head_dim * bits // 8, head_dim // BLOCK
    return QuantizedKV(zeros(elements), zeros(elements), zeros(scales), zeros(scales))


def _check_cache(cache, written: bool):
    """The sizes of one layer's cache: (num_pages, page_size, Hkv, D, bits, addresses and
    strides of elements and of scales as the library takes them)."""
    if not isinstance(cache, tuple) or len(cache) != 4 or not all(isinstance(t, torch.Tensor) for t in cache):
        raise ValueError("cache must be a QuantizedKV (or such a tuple) of four tensors")
    K, V, Ks, Vs = cache
    for t in (K, V, Ks, Vs):
        if t.dtype is not torch.uint8 or t.dim() != 4:
            raise ValueError("a quantized cache is four tensors of uint8 [pages, page_size, Hkv, bytes] (got "
                             f"{t.dtype} {tuple(t.shape)})")
    if K.shape != V.shape or Ks.shape != Vs.shape or K.shape[:3] != Ks.shape[:3]:
        raise ValueError(f"cache shapes differ: elements {tuple(K.shape)}, {tuple(V.shape)}, scales "
                         f"{tuple(Ks.shape)}, {tuple(Vs.shape)}")
    num_pages, page_size, Hkv, width = K.shape
    D = BLOCK * Ks.shape[3]
    if D not in (32, 64, 128) or width * 8 not in (4 * D, 8 * D) or Hkv < 1 or page_size < 1:
        raise ValueError(f"elements {tuple(K.shape)} and scales {tuple(Ks.shape)} are no cache of 4 or 8 bits with "
                         "heads of 32, 64 or 128")
    for a, b, unit, what in ((K, V, 16, "elements"), (Ks, Vs, D // BLOCK, "scales")):
        st = a.stride()
        if st != b.stride():
            raise ValueError(f"{what} of K and V must have the same strides (got {tuple(st)}, {tuple(b.stride())})")
        if not a.numel():
            continue
        if st[3] != 1 and a.shape[3] > 1 or any(x % unit for x in st[:3]) or (a.data_ptr() | b.data_ptr()) % unit:
            raise ValueError(f"{what} of strides {tuple(st)} are not rows of bytes on {unit}-byte boundaries")
        if written:
            if any(s == 0 and n > 1 for s, n in zip(st, a.shape)):
                raise ValueError("cache rows overlap (a stride of 0)")
            if a.data_ptr() == b.data_ptr():
                raise ValueError(f"{what} of K and V are the same memory")
    (cs, ss) = (_lib.layout(t.stride()[:3] + (1,))[0] for t in (K, Ks))
    return num_pages, page_size, Hkv, D, 2 * BLOCK * width // D // 8, (
        K.data_ptr(), V.data_ptr(), cs, Ks.data_ptr(), Vs.data_ptr(), ss)


def append_quantized_kv(
    K: torch.Tensor,
    V: torch.Tensor,
    cache: QuantizedKV,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_seqlen: int = None,
) -> torch.Tensor:
    """append_paged_kv with the rows quantised as they are written.

    K, V: packed fp16 or bf16 [T, Hkv, D].  Per 32 elements the scale is the smallest
    power of two s (at least 2^-126) whose 1.75 * 2^T * s (T = 2 in 4 bits, 8 in 8)
    reaches the largest magnitude, and no more than what keeps every element in the
    rows' range; elements are x / s rounded to nearest, ties to the even code, and
    end at the format's largest (6, 448).  A block with an infinity or a NaN is NaN.
    Positions, pages and lengths are append_paged_kv's; returns the lengths
    afterwards, int32 [B] on the device."""
    new = _lib.calls().quant_append(K, V, cache, page_table, context_lens, cu_seqlens, max_seqlen)
    if new is not None:
        return new
    num_pages, page_size, Hkv, D, bits, at = _check_cache(cache, written=True)
    assert K.dtype in _SUPPORTED and V.dtype == K.dtype, f"Inputs must be fp16 or bf16 (got {K.dtype}, {V.dtype})"
    idx = _device_index(K, V, *cache)
    _no_grad(K, V)
    device = K.device
    if K.dim() != 3 or K.shape != V.shape or tuple(K.shape[1:]) != (Hkv, D):
        raise ValueError(f"rows {tuple(K.shape)}, {tuple(V.shape)} incompatible with a cache of {Hkv} heads of {D}")
    T = K.shape[0]
    ctx = _lengths(context_lens, device)
    B = ctx.shape[0]
    ms, cu = _rows(T, B, cu_seqlens, max_seqlen, device)
    pt = _table(page_table, B, device)
    K, k, ks = _rows16(K)
    V, v, vs = _rows16(V)
    new = torch.empty_like(ctx)
    _launch(idx, "qattn_quant_append", _lib.lib().qattn_quant_append,
            k, ks, v, vs, *at, pt.data_ptr(), pt.shape[1], num_pages, page_size, ctx.data_ptr(), new.data_ptr(),
            _lib.ptr(cu), B, ms, T, Hkv, D, _dtype_code(K), bits)
    return new


def read_quantized_kv(
    cache: QuantizedKV,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_seqlen: int = None,
    total_tokens: int = None,
    dtype: torch.dtype = torch.float16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of the cache in 16 bits: row i of sequence s is its position starts[s] + i.

    cu_seqlens: packed offsets of the rows (None: one row per sequence); max_seqlen as
    everywhere; total_tokens: rows of the result, by default cu_seqlens[-1] (read on
    the host: pass both for graph capture).  A position that is negative, has no
    column or whose page lies outside the cache reads as zeros.  Rows that belong to
    no sequence, a sequence's rows past max_seqlen and all rows of one whose offsets
    descend or end past total_tokens are not written: they hold whatever the memory
    held, NaN perhaps.  Values are exact in bf16, and in fp16 where they lie in its
    range (as those written from fp16 rows do; larger ones become infinities).
    Returns K, V [total_tokens, Hkv, D]."""
    out = _lib.calls().quant_read(cache, page_table, starts, cu_seqlens, max_seqlen, total_tokens, dtype)
    if out is not None:
        return out
    num_pages, page_size, Hkv, D, bits, at = _check_cache(cache, written=False)
    if dtype not in _SUPPORTED:
        raise ValueError(f"dtype must be fp16 or bf16 (got {dtype})")
    idx = _device_index(*cache)
    device = cache.K.device
    start = _lengths(starts, device)
    B = start.shape[0]
    ms, cu = _rows(B, B, cu_seqlens, max_seqlen, device)
    T = B if cu is None else max(int(cu_seqlens[-1]), 0) if total_tokens is None else operator.index(total_tokens)
    if not 0 <= T < 2**31 or (cu is None and total_tokens not in (None, B)):
        raise ValueError(f"total_tokens must be the number of rows (got {total_tokens}, {T} rows, {B} sequences)")
    pt = _table(page_table, B, device)
    K, V = (torch.empty(T, Hkv, D, dtype=dtype, device=device) for _ in range(2))
    st = _lib.layout(K.stride())[0]
    _launch(idx, "qattn_quant_read", _lib.lib().qattn_quant_read,
            *at, pt.data_ptr(), pt.shape[1], num_pages, page_size, start.data_ptr(), K.data_ptr(), st, V.data_ptr(),
            st, _lib.ptr(cu), B, ms, T, Hkv, D, _dtype_code(K), bits)
    return K, V


def prefix_attention_quantized(
    Q: torch.Tensor,
    cache: QuantizedKV,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_seqlen: int = None,
    return_lse: bool = True,
):
    """prefix_attention_paged over a quantised cache: every query token of sequence s
    attends the values that positions 0 .. context_lens[s] - 1 stand for.

    Q: packed fp16 or bf16 [T, Hq, D], the cache's Hkv dividing Hq; page_table,
    context_lens, cu_seqlens, max_seqlen and the result are prefix_attention_paged's.
    The values are exact in the products; with fp16 queries they have to lie in fp16's
    range, as those written from fp16 rows do.  The elements span less than 64 GiB, the
    scales less than 2^32 rows (QAttnError otherwise).  A block whose scale is no number
    makes the rows that attend it NaN."""
    out = _lib.calls().quant_paged(Q, cache, page_table, context_lens, cu_seqlens, max_seqlen, return_lse)
    if out is not None:
        return out
    num_pages, page_size, Hkv, D, bits, at = _check_cache(cache, written=False)
    assert Q.dtype in _SUPPORTED, f"Inputs must be fp16 or bf16 (got {Q.dtype})"
    idx = _device_index(Q, *cache)
    _no_grad(Q)
    device = Q.device
    if Q.dim() != 3 or Q.shape[2] != D or Q.shape[1] % Hkv != 0 or Q.shape[1] < 1:
        raise ValueError(f"Q {tuple(Q.shape)} incompatible with a cache of {Hkv} heads of {D}")
    T, Hq, _ = Q.shape
    ctx = _lengths(context_lens, device)
    B = ctx.shape[0]
    ms, cu = _rows(T, B, cu_seqlens, max_seqlen, device)
    pt = _table(page_table, B, device)
    Q, q, qs = _rows16(Q)
    O, o, os_ = _out_like(Q)
    LSE = torch.empty(T, Hq, dtype=torch.float32, device=device) if return_lse else None
    L = _lib.lib()
    cols = pt.shape[1]
    ws_bytes = L.qattn_prefix_quant_workspace_bytes(B, ms, T, Hq, Hkv, D, cols, page_size, bits)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    _launch(idx, "qattn_prefix_quant_fwd", L.qattn_prefix_quant_fwd,
            q, qs, *at, pt.data_ptr(), cols, num_pages, page_size, ctx.data_ptr(), o, os_, _lib.ptr(LSE),
            None if LSE is None else _lib.layout(LSE.stride())[0], _lib.ptr(cu), B, ms, T, Hq, Hkv, D,
            1.0 / math.sqrt(D), _dtype_code(Q), bits, _lib.ptr(ws), ws_bytes)
    return (O, LSE) if return_lse else O
