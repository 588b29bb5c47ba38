"""Rows written into fp8 pages, and read back: the quantized caches that :func:`verify_attention` and
:func:`latent_verify_attention` read (``csrc/kv_pages.hip``).

A cache is ``[blocks, page, heads, D]`` ``float8_e4m3fn`` (any strides with a unit one over ``D``) with fp32 scales
``[blocks, heads]``. A page's scale is a power of two: e4m3 is a floating format, so the values' relative error is the same at
any scale, each is rounded once, and a scale that grows as a page fills moves the page's earlier rows without rounding
them again (but for those below e4m3's normal range).

A verify round keeps its rows at 16 bits (``k_new`` / ``v_new``) and writes the accepted ones after the walk, straight to
their chain slots: rejected rows touch neither a page nor its scale. A latent cache is the same with one head and no values.
"""

from __future__ import annotations

from typing import Optional

import torch

from eagle_harness.kernels import _native


_ROW_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _half(what: str, name: str, rows: torch.Tensor, cache: torch.Tensor, scale: torch.Tensor, device) -> tuple:
    """Checks keys or values; the strides of rows (token, head), cache (block, slot, head) and scales (block, head)."""
    if cache.dtype != torch.float8_e4m3fn:
        raise _native.NotCovered(f"{what}: {name}_cache must be float8_e4m3fn, got {cache.dtype}")
    row, page, scales, (blocks, _, heads, _), have = rows.stride(), cache.stride(), scale.stride(), cache.shape, scale.shape
    if row[2] != 1 or page[3] != 1:
        raise _native.NotCovered(f"{what}: {name} rows and cache must have a unit stride over the head dim")
    if scale.dtype != torch.float32 or len(have) != 2 or have[0] < blocks or have[1] < heads:
        raise ValueError(f"{what}: the {name} scales must be fp32 [blocks >= {blocks}, heads >= {heads}], got "
                         f"{scale.dtype} {tuple(have)}")
    if rows.device != device or cache.device != device or scale.device != device:
        raise ValueError(f"{what}: {name} rows, cache and scales must be on one device")
    return row, page, scales


def _pages_args(what: str, key: torch.Tensor, value: Optional[torch.Tensor], key_cache: torch.Tensor,
                value_cache: Optional[torch.Tensor], k_scale: torch.Tensor, v_scale: Optional[torch.Tensor],
                block_table: torch.Tensor) -> tuple:
    """Checks what writing and reading share; the struct's fields up to its tables, and (heads, dim, page, blocks)."""
    if (value is None) != (value_cache is None) or (value is None) != (v_scale is None):
        raise ValueError(f"{what}: value, value_cache and v_scale go together")
    rows, cache = key.shape, key_cache.shape
    if len(rows) != 3 or len(cache) != 4 or (value is not None and (value.shape != rows or value_cache.shape != cache)):
        raise ValueError(f"{what}: rows must be [tokens, heads, D] and caches [blocks, page, heads, D], values like keys")
    blocks, page, heads, dim = cache
    if rows[1] != heads or rows[2] != dim:
        raise ValueError(f"{what}: rows of {tuple(rows[1:])} do not fit a cache of {tuple(cache[2:])}")
    if key.dtype not in _ROW_DTYPES:
        raise _native.NotCovered(f"{what}: rows must be bf16, fp16 or fp32, got {key.dtype}")
    if value is not None and value.dtype != key.dtype:
        raise _native.NotCovered(f"{what}: key is {key.dtype} but value is {value.dtype}")
    device = key.device
    k, kc, ks = _half(what, "key", key, key_cache, k_scale, device)
    v, vc, vs = _NO_VALUES if value is None else _half(what, "value", value, value_cache, v_scale, device)
    if block_table.dim() != 2 or block_table.device != device:
        raise ValueError(f"{what}: the block table must be [requests, blocks] on the rows' device")
    fields = (key.data_ptr(), _native.ptr(value), k[0], k[1], v[0], v[1], key_cache.data_ptr(), _native.ptr(value_cache), kc[0],
              kc[1], kc[2], vc[0], vc[1], vc[2], k_scale.data_ptr(), _native.ptr(v_scale), ks[0], ks[1], vs[0], vs[1])
    return fields, (heads, dim, page, blocks)


_NO_VALUES = ((0, 0), (0, 0, 0), (0, 0))


def write_kv_pages(
    key: torch.Tensor,
    value: Optional[torch.Tensor],
    key_cache: torch.Tensor,
    value_cache: Optional[torch.Tensor],
    k_scale: torch.Tensor,
    v_scale: Optional[torch.Tensor],
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    *,
    max_query_len: int,
    idx_mapping: Optional[torch.Tensor] = None,
    path: Optional[torch.Tensor] = None,
    path_len: Optional[torch.Tensor] = None,
) -> None:
    """Quantizes rows into the pages behind each request's context, in place.

    ``key`` / ``value`` ``[tokens, heads, D]`` (bf16 / fp16 / fp32; ``value`` None for a latent cache): request ``b``'s rows are
    ``query_start_loc[b] ..``, at most ``max_query_len`` of them. Row ``j`` goes to position ``context_lens[b] + j`` of
    ``block_table[b]``. With ``path [slots, W]`` / ``path_len [slots]`` and ``idx_mapping [requests]`` (a
    :class:`~eagle_harness.vllm.verify_layout.TreeStore`'s, after the walk), position ``context_lens[b] + j`` takes row
    ``path[slot, j]`` for ``j < path_len[slot]``: the accepted rows alone, in chain order.

    The scale of a page that rows go to becomes the least power of two ``s`` with ``amax <= 448 s`` over them; a page that
    keeps earlier positions (below the context) keeps its scale if that is larger, and has them re-encoded if it is smaller.
    Positions behind a request's last row keep their bytes. Infinities saturate (at 448 times the scale) and do not
    count in ``amax``; a page of nothing else but zeros gets a scale of 1. A page belongs to one request. Rows whose page the table lacks, or names outside the cache, are not written, and neither is a
    path entry that names no row of its request; a page that no row goes to keeps its scale.
    """
    pages, (heads, dim, page, blocks) = _pages_args("write_kv_pages", key, value, key_cache, value_cache, k_scale, v_scale,
                                                    block_table)
    if 0 in pages:  # a stride: an expanded view, or a size of one
        for name, t in (("key_cache", key_cache), ("value_cache", value_cache), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
                raise ValueError(f"write_kv_pages: {name} is an expanded view: every page and head needs its own storage")
    num_reqs = query_start_loc.shape[0] - 1
    requests, max_blocks = block_table.shape
    if requests < num_reqs or context_lens.shape[0] < num_reqs:
        raise ValueError(f"write_kv_pages: block_table and context_lens must have {num_reqs} rows")
    if (path is None) != (path_len is None) or (path is not None and (idx_mapping is None or path.dim() != 2)):
        raise ValueError("write_kv_pages: path [slots, W], path_len [slots] and idx_mapping go together")
    device, width, slots = key.device, 0, 0
    if path is None:
        idx_mapping = None
    else:
        slots, width = path.shape
        slots = min(slots, path_len.shape[0])
        if idx_mapping.shape[0] < num_reqs:
            raise ValueError(f"write_kv_pages: idx_mapping must have {num_reqs} entries")
    for t in (context_lens, query_start_loc, path, path_len, idx_mapping):
        if t is not None and t.device != device:
            raise ValueError("write_kv_pages: every table must be on the rows' device")
    itab = _native.itab
    args = _native.WriteKvArgs(
        *pages, itab(block_table), itab(context_lens), itab(query_start_loc), itab(idx_mapping), itab(path), itab(path_len),
        key.shape[0], num_reqs, heads, dim, page, max_blocks, blocks, max_query_len, width, slots,
        _native.dtype_code(key.dtype))
    _native.launch("eagle4_write_kv_pages", args, device)


def read_kv_pages(
    key_cache: torch.Tensor,
    value_cache: Optional[torch.Tensor],
    k_scale: torch.Tensor,
    v_scale: Optional[torch.Tensor],
    block_table: torch.Tensor,
    start_loc: torch.Tensor,
    key_out: torch.Tensor,
    value_out: Optional[torch.Tensor],
    *,
    max_len: int,
) -> None:
    """Gathers the first ``start_loc[b + 1] - start_loc[b]`` (at most ``max_len``) positions of every request from fp8 pages
    into rows ``start_loc[b] ..`` of ``key_out`` / ``value_out`` ``[tokens, heads, D]`` (bf16 / fp16 / fp32): code times scale,
    rounded once. Rows behind the last request's are left alone; a position whose page the table lacks, or names outside
    the cache, reads as zeros."""
    pages, (heads, dim, page, blocks) = _pages_args("read_kv_pages", key_out, value_out, key_cache, value_cache, k_scale,
                                                    v_scale, block_table)
    num_reqs = start_loc.shape[0] - 1
    if block_table.shape[0] < num_reqs or start_loc.device != key_out.device:
        raise ValueError(f"read_kv_pages: block_table must have {num_reqs} rows, start_loc be on the rows' device")
    args = _native.ReadKvArgs(*pages, _native.itab(block_table), _native.itab(start_loc), key_out.shape[0], num_reqs, heads, dim,
                              page, block_table.shape[1], blocks, max_len, _native.dtype_code(key_out.dtype))
    _native.launch("eagle4_read_kv_pages", args, key_out.device)
