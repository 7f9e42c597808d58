"""A paged K/V cache around tree verification: attending it, filling it, keeping
the accepted path, copying pages.

The cache layout is build_paged_kv's: K_cache / V_cache [pages, page_size, Hkv,
D] and a page_table [B, max_pages] of int32 physical pages; position p of
sequence s is slot p % page_size of page page_table[s, p // page_size], and
context_lens[s] rows of it are filled.  compact_paged_kv and copy_kv_pages also
take the caches of all layers in one tensor, [layers, pages, page_size, Hkv, D]
(a layer's slice is the cache of the other calls).  Which pages a sequence owns
is the business of whoever fills the page table; no call here allocates or frees
pages.

A serving step over these calls, every tensor on the GPU (such a step can be
captured in a graph):

    # prompt: causal attention within it, its rows into the pages
    O = prompt_attention(Q, K, V, cu, max_seqlen)
    lens = append_paged_kv(K, V, K_cache, V_cache, table, lens, cu, max_seqlen)
    # decode: one token per sequence
    lens = append_paged_kv(k, v, K_cache, V_cache, table, lens)
    O, _ = prefix_attention_paged(q, K_cache, V_cache, table, lens)
    # verify a draft tree: context and tree, merged; its rows behind the context
    Oc, Lc = prefix_attention_paged(q, K_cache, V_cache, table, lens, cu, max_seqlen)
    Ot, Lt = ragged_attention_with_lse(q, k, v, cu, b, depth, max_seqlen)
    O = fused_lse_merge(...)
    append_paged_kv(k, v, K_cache, V_cache, table, lens, cu, max_seqlen)
    # keep the accepted path
    lens = compact_paged_kv(K_caches, V_caches, table, lens, accepted)

The calls run on torch's current stream, take contexts, offsets and page tables
on the host too (a copy each call, of what they hold at the call; not while a
graph is captured), and serve inference: tensors that ask for gradients are
refused while autograd records, those with tangents always.
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .ragged_attn import (_SUPPORTED, _check_dtypes, _device_index, _dtype_code, _integers, _launch, _no_grad,
                          _offsets, _out_like, _rows16, _to_device, _vec_ok)


def _int32(t: torch.Tensor, device) -> torch.Tensor:
    if t.dtype is torch.int32 and t.device == device and t.is_contiguous():
        return t
    return _to_device(_integers(t), device, in_graph=False)


def _check_caches(K_cache, V_cache, dims: Tuple[int, ...]) -> tuple:
    """Caches that a call writes in place: no copy can stand in for them.
    Returns their addresses and 5 strides {layer, page, slot, head, dim} each."""
    if K_cache.dtype is torch.uint8:
        return _check_bytes(K_cache, V_cache, dims)
    if K_cache.dim() not in dims or K_cache.shape != V_cache.shape:
        raise ValueError(f"caches must be {' or '.join(f'{d}-D' for d in dims)} and of one shape (got "
                         f"{tuple(K_cache.shape)}, {tuple(V_cache.shape)})")
    if K_cache.dtype not in _SUPPORTED or V_cache.dtype != K_cache.dtype:
        raise AssertionError(f"Inputs must be fp16 or bf16 (got {K_cache.dtype}, {V_cache.dtype})")
    (ks, k_ok), (vs, v_ok) = _lib.cache_layout(K_cache.stride()), _lib.cache_layout(V_cache.stride())
    k, v = K_cache.data_ptr(), V_cache.data_ptr()
    if (not k_ok or not v_ok or (k | v) & 15 or k == v) and K_cache.numel():
        for c in (K_cache, V_cache):
            if not _vec_ok(c):
                raise ValueError(f"cache of shape {tuple(c.shape)} and strides {tuple(c.stride())} is not writable as "
                                 "16-byte rows (unit last stride, 8-element aligned strides, 16-byte aligned base)")
            if any(st == 0 and n > 1 for st, n in zip(c.stride(), c.shape)):
                raise ValueError("cache rows overlap (a stride of 0)")
        if k == v:
            raise ValueError("K_cache and V_cache are the same memory")
    return k, ks, v, vs


def _check_bytes(K_cache, V_cache, dims: Tuple[int, ...]) -> tuple:
    """_check_caches for caches of bytes (a quantised cache's elements, or its scales)."""
    if K_cache.dim() not in dims or K_cache.shape != V_cache.shape or V_cache.dtype is not torch.uint8:
        raise ValueError(f"caches must be {' or '.join(f'{d}-D' for d in dims)}, of one shape and type (got "
                         f"{tuple(K_cache.shape)}, {V_cache.dtype} {tuple(V_cache.shape)})")
    width = K_cache.shape[-1]
    for c in (K_cache, V_cache):
        if c.stride(-1) != 1 and width > 1:
            raise ValueError(f"cache rows of strides {tuple(c.stride())} are no runs of bytes")
        if any(st == 0 and n > 1 for st, n in zip(c.stride(), c.shape)):
            raise ValueError("cache rows overlap (a stride of 0)")
    k, v = K_cache.data_ptr(), V_cache.data_ptr()
    if k == v and K_cache.numel():
        raise ValueError("K_cache and V_cache are the same memory")
    ks, vs = (_lib.cache_layout(c.stride()[:-1] + (1,))[0] for c in (K_cache, V_cache))
    return k, ks, v, vs


def _cache_code(cache) -> int:
    return _lib.DTYPE_U8 if cache.dtype is torch.uint8 else _dtype_code(cache)


def _table(page_table, B: int, device) -> torch.Tensor:
    if page_table.dim() != 2 or page_table.shape[0] < B:
        raise ValueError(f"page_table must be [B, max_pages] with B >= {B} (got {tuple(page_table.shape)})")
    return _int32(page_table, device)


def _lengths(context_lens, device) -> torch.Tensor:
    if context_lens.dim() != 1:
        raise ValueError(f"context_lens must be [B] (got {tuple(context_lens.shape)})")
    return _int32(context_lens, device)


def _rows(T: int, B: int, cu_seqlens, max_seqlen, device):
    """max_seqlen and the device offsets of packed rows; without offsets row s is sequence s's."""
    if cu_seqlens is None:
        if T != B:
            raise ValueError(f"without cu_seqlens there is one row per sequence (got {T} rows, {B} sequences)")
        return 1, None
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] != B + 1:
        raise ValueError(f"cu_seqlens must have {B + 1} entries (got {tuple(cu_seqlens.shape)})")
    return _offsets(cu_seqlens, device, max_seqlen)


def prefix_attention_paged(
    Q: torch.Tensor,
    K_cache: torch.Tensor,
    V_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_seqlen: int = None,
    return_lse: bool = True,
):
    """Attention of query tokens over their sequence's context in a paged cache:
    prefix_attention for pages, with a context length per sequence.

    Q: packed [T, Hq, D]; K_cache, V_cache: [pages, page_size, Hkv, D], Hkv
    dividing Hq; page_table [B, max_pages]; context_lens [B].  Every query token
    of sequence s attends positions 0 .. context_lens[s] - 1 (those that the
    table has columns for), not itself: append its row first, or merge another
    block by its LSE.  The lengths stay on the device, so the kernel is chosen by
    the table's width: columns past the longest context cost up to 5 us of a
    decode step's 8 to 30.  A cache spans less than 64 GiB, a layer's slice of one
    with the layers side by side in each page as much as all of them (QAttnError
    otherwise; the calls that move rows take any).

    cu_seqlens None: one token per sequence (a decode step); otherwise the packed
    offsets of the query tokens (draft trees, prompt chunks), max_seqlen as
    everywhere.  A page outside the cache removes its keys; a query without any
    gets 0 and an LSE of -inf.  Rows of Q that belong to no sequence are not
    computed.  Returns O [T, Hq, D] (and LSE [T, Hq] fp32, natural log, if
    return_lse)."""
    out = _lib.calls().paged(Q, K_cache, V_cache, page_table, context_lens, cu_seqlens, max_seqlen, return_lse)
    if out is not None:
        return out
    assert K_cache.shape == V_cache.shape, "K and V cache shapes must match"
    _check_dtypes(Q, K_cache, V_cache)
    idx = _device_index(Q, K_cache, V_cache)
    _no_grad(Q, K_cache, V_cache)
    device = Q.device
    if Q.dim() != 3 or K_cache.dim() != 4:
        raise ValueError(f"expected Q [T, Hq, D] and caches [pages, page_size, Hkv, D] (got {tuple(Q.shape)}, "
                         f"{tuple(K_cache.shape)})")
    T, Hq, D = Q.shape
    num_pages, page_size, Hkv, Dk = K_cache.shape
    if Dk != D or Hkv < 1 or Hq % Hkv != 0 or page_size < 1:
        raise ValueError(f"cache shape {tuple(K_cache.shape)} incompatible with Q {tuple(Q.shape)}")
    ctx = _lengths(context_lens, device)
    B = ctx.shape[0]
    ms, cu = _rows(T, B, cu_seqlens, max_seqlen, device)
    pt = _table(page_table, B, device)
    Q, q, qs = _rows16(Q)
    K_cache, k, ks = _rows16(K_cache)
    V_cache, v, vs = _rows16(V_cache)
    O, o, os_ = _out_like(Q)
    LSE = torch.empty(T, Hq, dtype=torch.float32, device=device) if return_lse else None
    L = _lib.lib()
    cols = pt.shape[1]
    ws_bytes = L.qattn_prefix_paged_workspace_bytes(B, ms, T, Hq, Hkv, D, cols, page_size)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    _launch(idx, "qattn_prefix_paged_fwd", L.qattn_prefix_paged_fwd,
            q, qs, k, ks, v, vs, pt.data_ptr(), cols, num_pages, page_size, ctx.data_ptr(), o, os_, _lib.ptr(LSE),
            None if LSE is None else _lib.layout(LSE.stride())[0], _lib.ptr(cu), B, ms, T, Hq, Hkv, D,
            1.0 / math.sqrt(D), _dtype_code(Q), _lib.ptr(ws), ws_bytes)
    return (O, LSE) if return_lse else O


def append_paged_kv(
    K: torch.Tensor,
    V: torch.Tensor,
    K_cache: torch.Tensor,
    V_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_seqlen: int = None,
) -> torch.Tensor:
    """Store new K/V rows behind each context, in place: row i of sequence s goes
    to position context_lens[s] + i.

    K, V: packed [T, Hkv, D]; cu_seqlens as in prefix_attention_paged (None: one
    row per sequence).  Returns the lengths afterwards, int32 [B] on the device;
    context_lens itself stays (rows behind a context do not count, so storing a
    draft tree and dropping the result leaves the context as it was).  A
    position that the table has no column for takes no row and does not count; a
    row whose page lies outside the cache is dropped.  A sequence with a negative
    length is passed over.  The written pages must be the sequence's own."""
    new = _lib.calls().append(K, V, K_cache, V_cache, page_table, context_lens, cu_seqlens, max_seqlen)
    if new is not None:
        return new
    kc, kcs, vc, vcs = _check_caches(K_cache, V_cache, (4,))
    _check_dtypes(K_cache, K, V)
    idx = _device_index(K_cache, V_cache, K, V)
    _no_grad(K, V, K_cache, V_cache)
    device = K.device
    num_pages, page_size, Hkv, D = K_cache.shape
    T = K.shape[0]
    if K.dim() != 3 or K.shape != V.shape or K.shape[1:] != K_cache.shape[2:] or page_size < 1:
        raise ValueError(f"rows {tuple(K.shape)}, {tuple(V.shape)} incompatible with cache {tuple(K_cache.shape)}")
    ctx = _lengths(context_lens, device)
    B = ctx.shape[0]
    ms, cu = _rows(T, B, cu_seqlens, max_seqlen, device)
    pt = _table(page_table, B, device)
    K, k, ks = _rows16(K)
    V, v, vs = _rows16(V)
    new = torch.empty_like(ctx)
    _launch(idx, "qattn_kv_append", _lib.lib().qattn_kv_append,
            k, ks, v, vs, kc, kcs, vc, vcs, pt.data_ptr(), pt.shape[1], num_pages, page_size, ctx.data_ptr(),
            new.data_ptr(), _lib.ptr(cu), B, ms, T, Hkv, D, _dtype_code(K))
    return new


def compact_paged_kv(
    K_cache: torch.Tensor,
    V_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    accepted: torch.Tensor,
) -> torch.Tensor:
    """Keep the accepted path of a draft tree whose rows were appended behind the
    context, in place: the row of node accepted[s, j] (position context_lens[s] +
    accepted[s, j]) moves to position context_lens[s] + j, in every layer.

    K_cache, V_cache: [layers, pages, page_size, Hkv, D] or one layer's [pages,
    page_size, Hkv, D], fp16, bf16 or the bytes of a quantised cache (its elements,
    or its scales); accepted: int32 [B, P], strictly increasing along a path
    (breadth-first order has ancestors before descendants), -1 behind its end; a
    path ends before the first entry that is not above its predecessor or that
    the table has no column for.  Returns the lengths afterwards, context plus
    path, int32 [B] on the device.  Pages of the moved positions must be the
    sequence's own."""
    new = _lib.calls().compact(K_cache, V_cache, page_table, context_lens, accepted)
    if new is not None:
        return new
    kc, kcs, vc, vcs = _check_caches(K_cache, V_cache, (4, 5))
    idx = _device_index(K_cache, V_cache)
    _no_grad(K_cache, V_cache)
    device = K_cache.device
    num_pages, page_size, Hkv, D = K_cache.shape[-4:]
    ctx = _lengths(context_lens, device)
    B = ctx.shape[0]
    if accepted.dim() != 2 or accepted.shape[0] != B or page_size < 1:
        raise ValueError(f"accepted must be [{B}, path length] (got {tuple(accepted.shape)})")
    pt, path = _table(page_table, B, device), _int32(accepted, device)
    new = torch.empty_like(ctx)
    layers = K_cache.shape[0] if K_cache.dim() == 5 else 1
    _launch(idx, "qattn_kv_compact", _lib.lib().qattn_kv_compact,
            kc, kcs, vc, vcs, layers, pt.data_ptr(), pt.shape[1], num_pages, page_size, ctx.data_ptr(),
            path.data_ptr(), path.shape[1], new.data_ptr(), B, Hkv, D, _cache_code(K_cache))
    return new


_Pages = Union[torch.Tensor, Sequence[int]]


def _whole(pages: Sequence[int]) -> list:
    try:
        return [operator.index(p) for p in pages]
    except TypeError as e:
        raise ValueError(f"pages must be integers ({e})") from None


def _page_lists(src, dst, num_pages: int, device):
    """Both lists on the device.  Lists on the host are checked: every page in
    the cache, no destination twice, none that is also a source."""
    src, dst = (_integers(t) if isinstance(t, torch.Tensor) else _whole(t) for t in (src, dst))
    shapes = [tuple(t.shape) if isinstance(t, torch.Tensor) else (len(t),) for t in (src, dst)]
    if len(shapes[0]) != 1 or shapes[0] != shapes[1]:
        raise ValueError(f"src_pages and dst_pages must be lists of one length (got {shapes[0]}, {shapes[1]})")
    s, d = (t if isinstance(t, list) else None if t.is_cuda else t.tolist() for t in (src, dst))
    for pages in (s, d):
        if pages is not None and any(not 0 <= p < num_pages for p in pages):
            raise ValueError(f"page outside [0, {num_pages})")
    if d is not None and len(set(d)) != len(d):
        raise ValueError("a page is the destination of two copies")
    if s is not None and d is not None:
        to = dict(zip(d, s))  # (a page copied onto itself stays as it is)
        if any(to.get(a, a) != a for a in s):
            raise ValueError("a page is the destination of one copy and the source of another")
    src, dst = (torch.tensor(t, dtype=torch.int32) if isinstance(t, list) else t for t in (src, dst))
    return _int32(src, device), _int32(dst, device)


def copy_kv_pages(K_cache: torch.Tensor, V_cache: torch.Tensor, src_pages: _Pages, dst_pages: _Pages) -> None:
    """Copy whole pages inside a cache, in place and in every layer: page
    dst_pages[i] takes page src_pages[i] of K and of V (the shared last page of a
    forked sequence, pages gathered to free others).

    K_cache, V_cache: [layers, pages, page_size, Hkv, D] or one layer's [pages,
    page_size, Hkv, D], fp16, bf16 or the bytes of a quantised cache.  The copies run
    side by side, so no page may be the destination of two or the destination of one
    and the source of another: lists on the host are checked for that (ValueError); of lists on the GPU,
    pairs with a page outside the cache are passed over, the rest is the
    caller's to keep."""
    if _lib.calls().copy(K_cache, V_cache, src_pages, dst_pages):
        return
    kc, kcs, vc, vcs = _check_caches(K_cache, V_cache, (4, 5))
    idx = _device_index(K_cache, V_cache)
    _no_grad(K_cache, V_cache)
    device = K_cache.device
    num_pages, page_size, Hkv, D = K_cache.shape[-4:]
    src, dst = _page_lists(src_pages, dst_pages, num_pages, device)
    if not src.shape[0] or not K_cache.numel():
        return
    layers = K_cache.shape[0] if K_cache.dim() == 5 else 1
    _launch(idx, "qattn_kv_copy_pages", _lib.lib().qattn_kv_copy_pages,
            kc, kcs, vc, vcs, layers, num_pages, page_size, src.data_ptr(), dst.data_ptr(), src.shape[0], Hkv, D,
            _cache_code(K_cache))
