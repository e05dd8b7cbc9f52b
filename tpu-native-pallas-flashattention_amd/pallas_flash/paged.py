"""Paged attention on MI355X: single-query attention over a page pool.

Drop-in for the reference's ``pallas_flash.paged`` (src/pallas_flash/paged.py).
Layout, as in the reference:

    k_pages / v_pages : [num_pages, num_kv_heads, page_size, head_dim]
    block_tables      : [batch, pages_per_seq]  int32  (logical -> physical page)
    context_lens      : [batch]                 int32  (valid tokens per sequence)

The HIP kernel reads the block table from device memory, so page gathering is
address arithmetic inside the kernel. Each KV head's pages are streamed once
for all query heads of its GQA group (the reference re-reads them per query
head). Table entries for logical pages at or past ``ceil(len / page_size)``
are never read, so ``-1`` padding is legal (the reference documents that its
unused entries must be valid indices because its DMA address is formed
regardless, paged.py:119-121).
"""

from __future__ import annotations

import operator
from typing import Optional, Sequence

import torch

from . import _lib
from ._shape import adapt, compute_dtype, decode_head_dim, restore, warn_copy


def paged_flash_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_tables,
    context_lens,
    *,
    sm_scale: Optional[float] = None,
    interpret: bool = False,
) -> torch.Tensor:
    """Single-query attention over a paged KV cache (reference: paged.py:102-192).

    Args:
        q: ``[batch, num_heads, 1, head_dim]``.
        k_pages, v_pages: ``[num_pages, num_kv_heads, page_size, head_dim]``.
        block_tables: ``[batch, pages_per_seq]`` integer table (cast to int32).
        context_lens: ``[batch]`` valid tokens per sequence (cast to int32). A
            sequence attends ``min(len, pages_per_seq * page_size)`` tokens;
            a non-positive length yields zeros.
        sm_scale: default ``1 / sqrt(head_dim)``.
        interpret: accepted for compatibility; ignored.

    Returns:
        ``[batch, num_heads, 1, head_dim]`` in q's dtype. Any head_dim up to
        256 that is a multiple of 8 (bfloat16/float16), or up to 128 that is
        a multiple of 4 (float32), is read in place; other head dims and
        mixed dtypes copy the pool padded/cast per call, with a one-time
        warning (``_shape``).
    """
    o = _lib.calls().paged(q, k_pages, v_pages, block_tables, context_lens, sm_scale)
    if o is not None:
        return o
    # paged.py:129-149
    if q.dim() != 4 or q.shape[2] != 1:
        raise ValueError(
            f"paged attention expects q of shape [batch, heads, 1, head_dim], got {tuple(q.shape)}")
    if k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    if k_pages.dim() != 4:
        raise ValueError("k_pages must be [num_pages, num_kv_heads, page_size, head_dim]")
    batch, num_heads, _, head_dim = q.shape
    num_pages, num_kv_heads, page_size, k_head_dim = k_pages.shape
    if k_head_dim != head_dim:
        raise ValueError("q and pages must share head_dim")
    if num_kv_heads == 0 or num_heads % num_kv_heads != 0:
        raise ValueError(
            f"num_heads ({num_heads}) must be a multiple of num_kv_heads ({num_kv_heads})")
    block_tables = torch.as_tensor(block_tables)
    context_lens = torch.as_tensor(context_lens)
    if block_tables.dim() != 2 or block_tables.shape[0] != batch:
        raise ValueError(
            f"block_tables must be [batch, pages_per_seq], got {tuple(block_tables.shape)}")
    if tuple(context_lens.shape) != (batch,):
        raise ValueError(f"context_lens must be [batch], got {tuple(context_lens.shape)}")
    if sm_scale is None:
        sm_scale = 1.0 / (head_dim ** 0.5)
    _lib.require_device(q, k_pages, v_pages)
    dev = q.device
    tables = block_tables.to(device=dev, dtype=torch.int32).contiguous()
    lens = context_lens.to(device=dev, dtype=torch.int32).contiguous()
    out_dtype = q.dtype
    cdt = compute_dtype(q, k_pages, v_pages)
    dp = decode_head_dim(head_dim, cdt)
    if dp != head_dim or k_pages.dtype != cdt or v_pages.dtype != cdt:
        warn_copy("paged_flash_attention", f"head_dim {head_dim} / dtypes {q.dtype}, {k_pages.dtype}, "
                  f"{v_pages.dtype} are not read in place")
    q, k_pages, v_pages = (adapt(x, cdt, dp).contiguous() for x in (q, k_pages, v_pages))
    o = torch.empty_like(q)
    if batch == 0:
        return restore(o, head_dim, out_dtype)
    args = _lib.PagedArgs(
        _lib.ptr(q), _lib.ptr(k_pages), _lib.ptr(v_pages), _lib.ptr(tables), _lib.ptr(lens),
        _lib.ptr(o), batch, num_heads, num_kv_heads, num_pages, page_size, dp,
        tables.shape[1], float(sm_scale), _lib.dtype_tag(q), None, 0)
    L = _lib.lib()
    ws_bytes = L.pf_paged_attn_workspace_min(args)
    ws = torch.empty(max(int(ws_bytes), 1), dtype=torch.uint8, device=dev)
    args.workspace = ws.data_ptr()
    args.workspace_bytes = ws.numel()
    with torch.cuda.device(dev):
        _lib.check(L.pf_paged_attn(args, _lib.stream_of(q)), "paged_flash_attention")
    return restore(o, head_dim, out_dtype)


def paged_flash_attention_prefix(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    prefix_table,
    prefix_len,
    block_tables,
    context_lens,
    *,
    sm_scale: Optional[float] = None,
) -> torch.Tensor:
    """Single-query attention of a batch whose sequences share a prefix
    (pf_paged_prefix_attn): each sequence attends the prefix's tokens and then
    its own. The result is that of ``paged_flash_attention`` with the prefix's
    tokens ahead of every sequence's; the prefix's K/V are read once for the
    batch instead of once per sequence (the reference's paged call,
    paged.py:102-192, knows no sharing). Two launches: where the prefix is short
    and the sequences few, ``paged_flash_attention`` over joined tables can be
    faster (5 us for 9).

    Args:
        q: ``[batch, num_heads, 1, head_dim]``.
        k_pages, v_pages: ``[num_pages, num_kv_heads, page_size, head_dim]``.
        prefix_table: ``[prefix_pages]`` integer table of the prefix's pages.
        prefix_len: tokens of the prefix: an int in ``[0, prefix_pages *
            page_size]`` (its last page need not be full), or a one-entry
            integer tensor on the device, which is not read back (the call stays
            capturable) and counts up to the table's reach. The work is divided
            for that reach: a prefix that fills little of a long table takes
            longer than with its length on the host (1000 tokens of 65536: 28 us
            for 15; of 2000: 15), so give a table near what it will hold.
        block_tables, context_lens: the sequences' own pages and tokens as
            ``paged_flash_attention`` takes them, the prefix not counted. A
            sequence without tokens at all yields zeros.
        sm_scale: default ``1 / sqrt(head_dim)``.

    Returns:
        ``[batch, num_heads, 1, head_dim]`` in q's dtype. Head dims and dtypes as
        ``paged_flash_attention``. No gradients: the result has no graph, whatever
        q and the pools require.
    """
    o = _lib.calls().prefix(q, k_pages, v_pages, prefix_table, prefix_len, block_tables, context_lens, sm_scale)
    if o is not None:
        return o
    if q.dim() != 4 or q.shape[2] != 1:
        raise ValueError(
            f"paged attention expects q of shape [batch, heads, 1, head_dim], got {tuple(q.shape)}")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [num_pages, num_kv_heads, page_size, head_dim] of one shape")
    batch, num_heads, _, head_dim = q.shape
    num_pages, num_kv_heads, page_size, k_head_dim = k_pages.shape
    if k_head_dim != head_dim or num_pages == 0 or page_size == 0:
        raise ValueError(f"q {tuple(q.shape)} does not match the pool {tuple(k_pages.shape)}")
    if num_kv_heads == 0 or num_heads == 0 or num_heads % num_kv_heads != 0:
        raise ValueError(f"num_heads ({num_heads}) must be a multiple of num_kv_heads ({num_kv_heads})")
    prefix_table, block_tables, context_lens = (torch.as_tensor(t) for t in (prefix_table, block_tables, context_lens))
    if prefix_table.dim() != 1:
        raise ValueError(f"prefix_table must be [prefix_pages], got {tuple(prefix_table.shape)}")
    if block_tables.dim() != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be [batch, pages_per_seq], got {tuple(block_tables.shape)}")
    if tuple(context_lens.shape) != (batch,):
        raise ValueError(f"context_lens must be [batch], got {tuple(context_lens.shape)}")
    for name, t in (("prefix_table", prefix_table), ("block_tables", block_tables), ("context_lens", context_lens)):
        # (an empty list makes a float tensor)
        if t.numel() > 0 and (t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool):
            raise ValueError(f"{name} must hold integers, got {t.dtype}")
    reach = prefix_table.shape[0] * page_size
    on_device = isinstance(prefix_len, torch.Tensor) and prefix_len.device.type != "cpu"
    if on_device:
        if prefix_len.numel() != 1 or prefix_len.dtype.is_floating_point or prefix_len.dtype == torch.bool:
            raise ValueError(f"prefix_len must be one integer, got {tuple(prefix_len.shape)} {prefix_len.dtype}")
    else:
        prefix_len = operator.index(prefix_len)
        if not 0 <= prefix_len <= reach:
            raise ValueError(f"prefix_len must be in [0, {reach}], got {prefix_len}")
    if sm_scale is None:
        sm_scale = 1.0 / (head_dim ** 0.5)
    _lib.require_device(q, k_pages, v_pages)
    dev = q.device
    prefix_table, tables, lens = (_lib.device_ints(t, dev) for t in (prefix_table, block_tables, context_lens))
    len_t = _lib.device_ints(prefix_len, dev).reshape(1) if on_device else None
    out_dtype = q.dtype
    cdt = compute_dtype(q, k_pages, v_pages)
    dp = decode_head_dim(head_dim, cdt)
    if dp != head_dim or k_pages.dtype != cdt or v_pages.dtype != cdt:
        warn_copy("paged_flash_attention_prefix", f"head_dim {head_dim} / dtypes {q.dtype}, {k_pages.dtype}, "
                  f"{v_pages.dtype} are not read in place")
    q, k_pages, v_pages = (adapt(x.detach(), cdt, dp).contiguous() for x in (q, k_pages, v_pages))
    o = torch.empty_like(q)
    if batch == 0:
        return restore(o, head_dim, out_dtype)
    args = _lib.PagedPrefixArgs(
        _lib.ptr(q), _lib.ptr(k_pages), _lib.ptr(v_pages), _lib.ptr(prefix_table), _lib.ptr(len_t), _lib.ptr(tables),
        _lib.ptr(lens), _lib.ptr(o), batch, num_heads, num_kv_heads, num_pages, page_size, dp, prefix_table.shape[0],
        reach if on_device else prefix_len, tables.shape[1], float(sm_scale), _lib.dtype_tag(q), None, 0)
    L = _lib.lib()
    with torch.cuda.device(dev):
        ws_bytes = L.pf_paged_prefix_attn_workspace_size(args)
        ws = torch.empty(max(int(ws_bytes), 1), dtype=torch.uint8, device=dev)
        args.workspace = ws.data_ptr()
        args.workspace_bytes = ws.numel()
        _lib.check(L.pf_paged_prefix_attn(args, _lib.stream_of(q)), "paged_flash_attention_prefix")
    return restore(o, head_dim, out_dtype)


def init_paged_cache(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
                     dtype=torch.float32, device=None):
    """Allocate an empty page pool ``(k_pages, v_pages)`` (paged.py:198-202)."""
    shape = (num_pages, num_kv_heads, page_size, head_dim)
    return (torch.zeros(shape, dtype=dtype, device=device),
            torch.zeros(shape, dtype=dtype, device=device))


def write_to_paged_cache(k_pages, v_pages, k, v, block_table, position, *, inplace: bool = True):
    """Write token K/V into the pages holding their positions
    (paged.py:205-223), on device (pf_paged_cache_write), in place by default.

    The reference writes one token of one sequence: ``k``/``v``
    ``[1, num_kv_heads, 1, head_dim]``, ``block_table`` ``[pages_per_seq]``,
    ``position`` an int. The same call also takes a batch: ``k``/``v``
    ``[batch, num_kv_heads, seq_len, head_dim]``, ``block_table``
    ``[batch, pages_per_seq]`` and ``position`` an int or ``[batch]``
    integers (row ``i`` of sequence ``b`` goes to position
    ``position[b] + i``). A row whose position falls outside the table, or
    whose table entry is not a page of the pool (e.g. ``-1`` padding), is not
    written (the reference's dynamic_update_slice would clamp it onto a valid
    slot).

    Returns the updated ``(k_pages, v_pages)``: with ``inplace=True``
    (default) the same tensors, written in place, so the reference's
    functional call pattern keeps working without a pool copy; with
    ``inplace=False`` written copies, the given pools left unchanged, as the
    reference's functional update leaves them (one pool-sized device copy
    per call: for callers that keep the pre-write pool, e.g. to roll back
    speculative tokens).
    """
    from .cache import _check_positions, _positions
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [num_pages, num_kv_heads, page_size, head_dim] of one shape")
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError("k and v must be [batch, num_kv_heads, seq_len, head_dim] of one shape")
    num_pages, hkv, page_size, d = k_pages.shape
    batch = k.shape[0]
    if k.shape[1] != hkv or k.shape[3] != d:
        raise ValueError(f"k {tuple(k.shape)} does not match the pool {tuple(k_pages.shape)}")
    if k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must share a dtype")
    table = torch.as_tensor(block_table)
    if table.dim() == 1:
        table = table.unsqueeze(0)
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"block_table must be [pages_per_seq] or [batch, pages_per_seq], got {tuple(table.shape)}")
    _check_positions(position, batch)
    _lib.require_device(k_pages, v_pages, k, v)
    if not inplace:
        k_pages, v_pages = (t.clone(memory_format=torch.contiguous_format) for t in (k_pages, v_pages))
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("the page pools are written in place and must be contiguous")
    dev = k_pages.device
    table = table.to(device=dev, dtype=torch.int32).contiguous()
    pos, stride = _positions(position, batch, dev)
    k = k.to(k_pages.dtype).contiguous()
    v = v.to(k_pages.dtype).contiguous()
    args = _lib.PagedWriteArgs(_lib.ptr(k), _lib.ptr(v), _lib.ptr(k_pages), _lib.ptr(v_pages), _lib.ptr(table),
                               _lib.ptr(pos), stride, batch, hkv, k.shape[2], num_pages, page_size, d,
                               table.shape[1], _lib.dtype_tag(k_pages))
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().pf_paged_cache_write(args, _lib.stream_of(k_pages)), "write_to_paged_cache")
    return k_pages, v_pages


def write_to_paged_cache_rope(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    block_table,
    position,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    rope_positions=None,
    sections: Optional[Sequence[int]] = None,
    seq_lens=None,
):
    """Rotate the new tokens' q and k and write k and v into their pages, in
    one launch (pf_rope_paged_cache_write): the part of a layer between its
    projections and ``paged_flash_attention``. The reference rotates first
    (model.py:340-341) and writes one token of one sequence (paged.py:205-223).

    Args:
        k_pages, v_pages: ``[num_pages, num_kv_heads, page_size, head_dim]``,
            written in place.
        q: ``[batch, num_heads, seq_len, head_dim]``, before RoPE.
        k, v: ``[batch, num_kv_heads, seq_len, head_dim]``, k before RoPE. All
            of one dtype; read with their own strides (views of one fused
            projection are not copied).
        block_table, position: as ``write_to_paged_cache``: row ``i`` of
            sequence ``b`` lands at position ``position[b] + i`` of its table;
            a row without a page there is not written.
        cos, sin: ``[rope_len, head_dim]`` tables (``precompute_rope``).
        rope_positions: the rotary positions where they are not the rows' own
            ``position[b] + i`` (several axes; tokens behind a shared prefix):
            integers ``[axes, seq_len]`` or ``[axes, batch, seq_len]`` as
            ``apply_rope_axes`` takes them. A row with one outside the tables
            writes nothing, its q is zero.
        sections: the rotated pairs of each axis (``apply_rope_axes``); several
            axes need ``rope_positions``.
        seq_lens: ``[batch]`` integers: rows at or past them are padding --
            nothing is written, q is zero. ``None``: all rows are tokens.

    Returns ``(q_rot, k_pages, v_pages)``: the rotated q, dense, and the pools.
    No gradients: the pools belong to inference.
    """
    q_rot = _lib.calls().rope_write(k_pages, v_pages, q, k, v, block_table, position, cos, sin, rope_positions,
                                    sections, seq_lens)
    if q_rot is not None:
        return q_rot, k_pages, v_pages
    from .cache import _check_positions
    from .rope_axes import (check_axis_positions, check_sections, check_tables, device_positions, rows_of, sections4,
                            strides3)
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [num_pages, num_kv_heads, page_size, head_dim] of one shape")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q must be [batch, num_heads, seq_len, head_dim], k and v [batch, num_kv_heads, seq_len, "
                         "head_dim] of one shape")
    num_pages, hkv, page_size, d = k_pages.shape
    batch, hq, seq, _ = q.shape
    if k.shape[1] != hkv or k.shape[3] != d or num_pages == 0 or page_size == 0:
        raise ValueError(f"k {tuple(k.shape)} does not match the pool {tuple(k_pages.shape)}")
    if q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.shape[3] != d:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must share batch, seq_len and head_dim")
    if hkv == 0 or hq == 0 or hq % hkv != 0:
        raise ValueError(f"num_heads ({hq}) must be a multiple of num_kv_heads ({hkv})")
    if any(t.dtype != k_pages.dtype for t in (v_pages, q, k, v)):
        raise ValueError("q, k, v and the pools must share a dtype")
    sections = check_sections(sections, d)
    check_tables(cos, sin, d)
    if rope_positions is not None:
        rope_positions = check_axis_positions(rope_positions, len(sections), batch, seq)
    elif len(sections) > 1:
        raise ValueError("several axes need rope_positions")
    table = torch.as_tensor(block_table)
    if table.dim() == 1:
        table = table.unsqueeze(0)
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"block_table must be [pages_per_seq] or [batch, pages_per_seq], got {tuple(table.shape)}")
    _check_positions(position, batch)
    if seq_lens is not None:
        seq_lens = torch.as_tensor(seq_lens)
        if tuple(seq_lens.shape) != (batch,) or seq_lens.dtype.is_floating_point or seq_lens.dtype == torch.bool:
            raise ValueError(f"seq_lens must be [batch] integers, got {tuple(seq_lens.shape)} {seq_lens.dtype}")
    _lib.require_device(k_pages, v_pages, q, k, v)
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("the page pools are written in place and must be contiguous")
    dev = k_pages.device
    q_rot = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if q_rot.numel() == 0:
        return q_rot, k_pages, v_pages
    q, k, v = (rows_of(t.detach()) for t in (q, k, v))
    table = _lib.device_ints(table, dev)
    pos, stride = _check_positions(position, batch)
    pos = _lib.device_ints(pos, dev)
    if seq_lens is not None:
        seq_lens = _lib.device_ints(seq_lens, dev)
    rope, rope_stride, i64 = None, (0, 0, 0), 0
    if rope_positions is not None:
        rope, rope_stride, i64 = device_positions(rope_positions, dev)
    cos, sin = (t.detach().to(device=dev, dtype=torch.float32).contiguous() for t in (cos, sin))
    args = _lib.RopePagedWriteArgs(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(q_rot), _lib.ptr(k_pages), _lib.ptr(v_pages), strides3(q),
        strides3(k), strides3(v), _lib.ptr(table), _lib.ptr(pos), stride, _lib.ptr(seq_lens), _lib.ptr(rope),
        (_lib.c_i64 * 3)(*rope_stride), i64, len(sections), sections4(sections), _lib.ptr(cos), _lib.ptr(sin),
        cos.shape[0], batch, hq, hkv, seq, num_pages, page_size, d, table.shape[1], _lib.dtype_tag(k_pages))
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().pf_rope_paged_cache_write(args, _lib.stream_of(k_pages)), "write_to_paged_cache_rope")
    return q_rot, k_pages, v_pages


__all__ = ["paged_flash_attention", "paged_flash_attention_prefix", "init_paged_cache", "write_to_paged_cache",
           "write_to_paged_cache_rope"]
