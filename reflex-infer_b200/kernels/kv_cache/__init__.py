"""Paged KV pool operations; same surface as the reference's ``kernels/kv_cache/__init__.py``.

* ``kv_paged_append``  : write new K/V rows at flat slots (``kv_cache/__init__.py:31-51``).
* ``kv_paged_lookup``  : gather pages into dense ``[B, H, max_ctx, D]`` with a zero tail
  (``kv_cache/__init__.py:54-71``).
* ``kv_paged_scatter`` : overwrite slots; the same operation as append
  (``kv_cache/__init__.py:74-90``).

Pool layout ``[num_blocks, num_heads, block_size, head_dim]``, ``slot = page*block_size + pos``
(``triton_kv_paged.py:9-15``). The caches are mutated in place.

Page bookkeeping (additive; the reference leaves it to its caller), all of it on the device, with
``ref_counts`` ``[num_blocks]`` int32 as its state (requests that hold a page, 0 = free):

* ``kv_fork``       : children share their parent's whole pages, take a page for a part-filled last one.
* ``kv_free``       : rows of the table give their pages up.
* ``kv_compact``    : the live pages move to the front of the pool.
* ``kv_copy_pages`` : the copies that fork and compact ask for (``PageMoves``), for all layers at once.
"""
from __future__ import annotations

from array import array
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from .. import _native as N


def _check_pool(name, k_cache, v_cache):
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"{name}: caches must both be [num_blocks, num_heads, block_size, head_dim]; "
                         f"got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError(f"{name}: k_cache and v_cache dtypes differ")
    if k_cache.stride() != v_cache.stride():
        raise ValueError(f"{name}: k_cache and v_cache must share one stride pattern")
    if k_cache.stride(3) != 1:
        raise ValueError(f"{name}: the head_dim axis of the caches must be contiguous")


def _write_slots(entry, name, k_in, v_in, k_cache, v_cache, slot_mapping):
    dev = N.require_cuda(name, k_in, v_in, k_cache, v_cache, slot_mapping)
    _check_pool(name, k_cache, v_cache)
    if k_in.dim() != 3 or v_in.shape != k_in.shape:
        raise ValueError(f"{name}: k_in and v_in must both be [N, num_heads, head_dim]")
    n, heads, dim = k_in.shape
    nb, ch, bs, cd = k_cache.shape
    if (heads, dim) != (ch, cd):
        raise ValueError(f"{name}: input heads/head_dim {(heads, dim)} do not match the cache {(ch, cd)}")
    if k_in.dtype != k_cache.dtype or v_in.dtype != k_cache.dtype:
        # torch's index_put_ refuses this too ("source and destination dtypes match")
        raise RuntimeError(f"{name}: input dtype {k_in.dtype} does not match cache dtype {k_cache.dtype}")
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != n:
        raise ValueError(f"{name}: slot_mapping must be [N]={n}, got {tuple(slot_mapping.shape)}")
    if slot_mapping.dtype != torch.int64:
        slot_mapping = slot_mapping.to(torch.int64)
    slot_mapping = slot_mapping.contiguous()
    if k_in.stride(2) != 1 or v_in.stride() != k_in.stride():
        k_in, v_in = k_in.contiguous(), v_in.contiguous()
    a = N.KvAppendArgs(
        k_in=N.ptr(k_in), v_in=N.ptr(v_in), k_cache=N.ptr(k_cache), v_cache=N.ptr(v_cache),
        slot_mapping=N.ptr(slot_mapping),
        n_tokens=n, num_kv_heads=heads, head_dim=dim, num_blocks=nb, block_size=bs,
        in_stride_n=k_in.stride(0), in_stride_h=k_in.stride(1),
        cache_stride_blk=k_cache.stride(0), cache_stride_h=k_cache.stride(1), cache_stride_pos=k_cache.stride(2),
        dtype=N.dtype_code(k_cache), stream=N.stream_handle(dev),
    )
    N.call(entry, a, dev)


def kv_paged_append(
    k_in: torch.Tensor,
    v_in: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    backend: Optional[str] = None,
) -> None:
    """Append new K, V into the paged KV cache (in place).

    ``k_in``/``v_in``: ``[N, num_heads, head_dim]``; ``slot_mapping``: ``[N]`` int64 flat
    slots. Slots must be distinct; a slot outside the pool is skipped.
    """
    N.check_backend(backend)
    _write_slots("rfx_kv_paged_append", "kv_paged_append", k_in, v_in, k_cache, v_cache, slot_mapping)


def kv_paged_lookup(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    max_ctx: int,
    *,
    backend: Optional[str] = None,
) -> tuple:
    """Gather K, V from the paged cache into dense ``[B, num_heads, max_ctx, head_dim]``
    tensors; positions at or beyond ``context_lens[b]`` are zero in both."""
    N.check_backend(backend)
    name = "kv_paged_lookup"
    dev = N.require_cuda(name, k_cache, v_cache, block_table, context_lens)
    _check_pool(name, k_cache, v_cache)
    if block_table.dim() != 2:
        raise ValueError(f"{name}: block_table must be [B, max_blocks]")
    B = context_lens.shape[0]
    if block_table.shape[0] != B:
        raise ValueError(f"{name}: block_table has {block_table.shape[0]} rows, context_lens {B}")
    if block_table.dtype != torch.int64:
        block_table = block_table.to(torch.int64)
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    if context_lens.dtype != torch.int32:
        context_lens = context_lens.to(torch.int32)
    context_lens = context_lens.contiguous()
    nb, heads, bs, dim = k_cache.shape
    max_ctx = int(max_ctx)
    k_out = torch.empty((B, heads, max_ctx, dim), dtype=k_cache.dtype, device=dev)
    v_out = torch.empty_like(k_out)
    a = N.KvLookupArgs(
        k_cache=N.ptr(k_cache), v_cache=N.ptr(v_cache), k_out=N.ptr(k_out), v_out=N.ptr(v_out),
        block_table=N.ptr(block_table), context_lens=N.ptr(context_lens),
        batch=B, num_kv_heads=heads, head_dim=dim, num_blocks=nb, block_size=bs,
        max_ctx=max_ctx, max_blocks=block_table.shape[1],
        cache_stride_blk=k_cache.stride(0), cache_stride_h=k_cache.stride(1), cache_stride_pos=k_cache.stride(2),
        bt_stride_b=block_table.stride(0),
        dtype=N.dtype_code(k_cache), stream=N.stream_handle(dev),
    )
    N.call("rfx_kv_paged_lookup", a, dev)
    return k_out, v_out


def kv_paged_scatter(
    k_updates: torch.Tensor,
    v_updates: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    backend: Optional[str] = None,
) -> None:
    """Overwrite specific slots (speculative decoding rollback, page compaction)."""
    N.check_backend(backend)
    _write_slots("rfx_kv_paged_scatter", "kv_paged_scatter", k_updates, v_updates, k_cache, v_cache, slot_mapping)


class PageMoves(NamedTuple):
    """Pages to copy: ``src[i]`` onto ``dst[i]`` (int64; a pair with -1 is none), the first ``rows[i]``
    positions (int32; ``None``: all of them), for the first ``count[0]`` pairs (int32; ``None``: for all)."""

    src: torch.Tensor
    dst: torch.Tensor
    rows: Optional[torch.Tensor] = None
    count: Optional[torch.Tensor] = None


_fork = N.Entry("rfx_kv_fork", N.KvForkArgs)
_free = N.Entry("rfx_kv_free", N.KvFreeArgs)
_compact = N.Entry("rfx_kv_compact", N.KvCompactArgs)
_copy = N.Entry("rfx_kv_copy_pages", N.KvCopyArgs)


def _check_table(name, block_table, ref_counts):
    if block_table.dim() != 2 or block_table.dtype != torch.int64:
        raise ValueError(f"{name}: block_table must be int64 [rows, max_blocks], "
                         f"got {block_table.dtype} {tuple(block_table.shape)}")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError(f"{name}: the entries of a block_table row must be contiguous")
    if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError(f"{name}: the rows of block_table overlap")
    if ref_counts.dim() != 1 or ref_counts.dtype != torch.int32 or not ref_counts.is_contiguous():
        raise ValueError(f"{name}: ref_counts must be contiguous int32 [num_blocks], "
                         f"got {ref_counts.dtype} {tuple(ref_counts.shape)}")
    if ref_counts.shape[0] == 0:
        raise ValueError(f"{name}: ref_counts is empty")


def _int32_vector(name, what, t, n=None):
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name}: {what} must be [{'n' if n is None else n}], got {tuple(t.shape)}")
    if t.dtype != torch.int32:
        if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
            raise ValueError(f"{name}: {what} must hold whole numbers, got {t.dtype}")
        t = t.clamp(-1, 2**31 - 1).to(torch.int32) if t.dtype == torch.int64 else t.to(torch.int32)
    return t.contiguous()


def kv_fork(
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    parents: torch.Tensor,
    ref_counts: torch.Tensor,
    block_size: int,
    *,
    backend: Optional[str] = None,
) -> Tuple[torch.Tensor, PageMoves]:
    """Child ``i`` continues row ``parents[i]`` of ``block_table``: returns ``(child_table, moves)``.

    A child shares its parent's whole pages (``ref_counts`` up by one each, in place). Where the parent's
    ``context_lens`` ends inside a page the child takes the lowest free page for itself, and ``moves``
    says which positions to copy there: give it to ``kv_copy_pages`` before the child's next token is
    appended. ``child_table`` is ``[n, max_blocks]`` int64, -1 behind the child's pages. Children take free
    pages in order; one for which none is left has ``moves.src >= 0`` and ``moves.dst < 0``, and it (and one
    whose parent is no row) gets a row of -1 and holds nothing. A parent may have any number of children;
    it keeps its own pages until ``kv_free``.

    ``ref_counts`` has to be true: every page that a parent's row names within its length counts 1 at least, and then no
    page of any row is handed out. A page that counts 0 is free: a whole one that a row names all the same may become another
    child's own page and be overwritten by its copy. Only the part-filled page that a child copies from is never handed
    out, whatever its count (0 becomes 1), so the copies of one call cannot meet.
    """
    N.check_backend(backend)
    name = "kv_fork"
    index = N.same_device(name, block_table, context_lens, parents, ref_counts)
    _check_table(name, block_table, ref_counts)
    if int(block_size) <= 0:
        raise ValueError(f"{name}: block_size must be positive, got {block_size}")
    batch, max_blocks = block_table.shape
    context_lens = _int32_vector(name, "context_lens", context_lens, batch)
    parents = _int32_vector(name, "parents", parents)
    n = parents.shape[0]
    child = block_table.new_empty((n, max_blocks))
    src, dst = block_table.new_empty(n), block_table.new_empty(n)
    rows = parents.new_empty(n)
    _fork(index, block_table.data_ptr(), context_lens.data_ptr(), parents.data_ptr(), ref_counts.data_ptr(),
          child.data_ptr(), src.data_ptr(), dst.data_ptr(), rows.data_ptr(),
          n, batch, max_blocks, block_table.stride(0), ref_counts.shape[0], int(block_size), N.stream_of(index))
    return child, PageMoves(src, dst, rows)


def kv_free(
    block_table: torch.Tensor,
    rows: torch.Tensor,
    ref_counts: torch.Tensor,
    *,
    backend: Optional[str] = None,
) -> None:
    """The given rows of ``block_table`` give up every page they name: the entries become -1 and the
    pages' ``ref_counts`` go down by one (in place). A row that is named twice or was freed before gives
    its pages up once; a row outside the table is skipped."""
    N.check_backend(backend)
    name = "kv_free"
    index = N.same_device(name, block_table, rows, ref_counts)
    _check_table(name, block_table, ref_counts)
    rows = _int32_vector(name, "rows", rows)
    _free(index, block_table.data_ptr(), rows.data_ptr(), ref_counts.data_ptr(), rows.shape[0], block_table.shape[0],
          block_table.shape[1], block_table.stride(0), ref_counts.shape[0], N.stream_of(index))


def kv_compact(
    block_table: torch.Tensor,
    ref_counts: torch.Tensor,
    *,
    backend: Optional[str] = None,
) -> Tuple[torch.Tensor, PageMoves]:
    """Moves the live pages to the front of the pool: returns ``(page_map, moves)``.

    With ``live`` pages in use, those at index ``live`` and behind go into the free pages below it, the
    last one into the first. ``block_table`` and ``ref_counts`` are rewritten in place; give ``moves`` to
    ``kv_copy_pages`` before the pool is read again. ``page_map`` ``[num_blocks]`` int64 holds every page's
    new index (-1: free), for tables other than this one; an entry of ``block_table`` that names a free
    page becomes -1, one outside the pool is left as it is.
    """
    N.check_backend(backend)
    name = "kv_compact"
    index = N.same_device(name, block_table, ref_counts)
    _check_table(name, block_table, ref_counts)
    num = ref_counts.shape[0]
    page_map = block_table.new_empty(num)
    src, dst = block_table.new_empty(num // 2 + 1), block_table.new_empty(num // 2 + 1)
    need = int(N.lib().rfx_kv_compact_workspace_bytes(num))
    words = ref_counts.new_empty(64 + need // 4)  # the number of moves stands in front of the scratch
    count = words[:1]
    _compact(index, block_table.data_ptr(), ref_counts.data_ptr(), page_map.data_ptr(), src.data_ptr(), dst.data_ptr(),
             count.data_ptr(), block_table.shape[0], block_table.shape[1], block_table.stride(0), num,
             words.data_ptr() + 256, need, N.stream_of(index))
    return page_map, PageMoves(src, dst, None, count)


def _layers(t):
    return [t] if isinstance(t, torch.Tensor) else list(t)


def _pointers(tensors):
    """The tensors' addresses as a C array."""
    return array("Q", [t.data_ptr() for t in tensors])


def kv_copy_pages(
    k_cache: Union[torch.Tensor, Sequence[torch.Tensor]],
    v_cache: Union[torch.Tensor, Sequence[torch.Tensor]],
    moves: PageMoves,
    *,
    k_scales: Union[None, torch.Tensor, Sequence[torch.Tensor]] = None,
    v_scales: Union[None, torch.Tensor, Sequence[torch.Tensor]] = None,
    backend: Optional[str] = None,
) -> None:
    """Copies pages inside the caches of one layer, or of all layers given as lists, in place.

    ``moves`` comes from ``kv_fork`` or ``kv_compact`` or is a ``PageMoves`` of one's own. All layers share
    one shape and stride pattern; int8 caches need their ``k_scales`` / ``v_scales`` ``[num_blocks, H_kv,
    block_size]``, which move along. A pair with an index outside the pool is skipped; positions from
    ``moves.rows[i]`` on are left as they are. Destinations must be distinct and none may be a source.
    """
    N.check_backend(backend)
    name = "kv_copy_pages"
    ks, vs = _layers(k_cache), _layers(v_cache)
    if len(ks) != len(vs) or not ks:
        raise ValueError(f"{name}: as many k as v caches are needed, at least one; got {len(ks)} and {len(vs)}")
    src, dst, rows, count = moves
    first = ks[0]
    index = N.same_device(name, first, src, dst, rows, count, *ks, *vs)
    shape, strides, dtype = first.shape, first.stride(), first.dtype
    if len(shape) != 4 or strides[3] != 1:
        raise ValueError(f"{name}: caches must be [num_blocks, num_heads, block_size, head_dim], the last axis contiguous; "
                         f"got {tuple(shape)}, strides {strides}")
    for t in ks + vs:
        if t is not first and (t.shape != shape or t.stride() != strides or t.dtype != dtype):
            raise ValueError(f"{name}: all caches must share one shape, stride pattern and dtype")
    if src.dtype != torch.int64 or dst.dtype != torch.int64 or src.dim() != 1 or dst.shape != src.shape:
        raise ValueError(f"{name}: moves.src and moves.dst must be int64 [n]")
    n = src.shape[0]
    src, dst = src.contiguous(), dst.contiguous()
    if rows is not None:
        rows = _int32_vector(name, "moves.rows", rows, n)
    if count is not None and (count.dtype != torch.int32 or count.numel() != 1):
        raise ValueError(f"{name}: moves.count must be one int32")
    L = len(ks)
    k_ptrs, v_ptrs = _pointers(ks), _pointers(vs)
    int8, k_scale_ptrs, v_scale_ptrs = 0, None, None
    if dtype == torch.int8:
        int8 = 1
        if k_scales is None or v_scales is None:
            raise ValueError(f"{name}: an int8 pool needs k_scales and v_scales")
        sk, sv = _layers(k_scales), _layers(v_scales)
        N.same_device(name, first, *sk, *sv)
        if len(sk) != L or len(sv) != L:
            raise ValueError(f"{name}: every layer needs its scales")
        for t in sk + sv:
            if t.dtype != torch.float32 or t.shape != shape[:3] or not t.is_contiguous():
                raise ValueError(f"{name}: scales must be contiguous float32 {list(shape[:3])}")
        k_scale_ptrs, v_scale_ptrs = _pointers(sk), _pointers(sv)
    _copy(index, k_ptrs.buffer_info()[0], v_ptrs.buffer_info()[0], k_scale_ptrs.buffer_info()[0] if int8 else 0,
          v_scale_ptrs.buffer_info()[0] if int8 else 0, src.data_ptr(), dst.data_ptr(),
          0 if rows is None else rows.data_ptr(), 0 if count is None else count.data_ptr(),
          L, n, shape[1], shape[3], shape[0], shape[2], strides[0], strides[1], strides[2],
          0 if int8 else N.dtype_code(first), int8, N.stream_of(index))


# The reference's surface; the page bookkeeping above is an addition, imported by name.
__all__ = [
    "kv_paged_append",
    "kv_paged_lookup",
    "kv_paged_scatter",
]
