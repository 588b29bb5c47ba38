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


def _check_pages(what: str, key: torch.Tensor, value: Optional[torch.Tensor], key_cache: torch.Tensor,
                 value_cache: Optional[torch.Tensor], k_scale: torch.Tensor, v_scale: Optional[torch.Tensor],
                 block_table: torch.Tensor) -> None:
    if (value is None) != (value_cache is None) or (value is None) != (v_scale is None):
        raise ValueError(f"{what}: value, value_cache and v_scale go together")
    if key.dim() != 3 or key_cache.dim() != 4 or (value is not None and (value.shape != key.shape
                                                                       or value_cache.shape != key_cache.shape)):
        raise ValueError(f"{what}: rows must be [tokens, heads, D] and caches [blocks, page, heads, D], values like keys")
    if key.shape[1:] != key_cache.shape[2:]:
        raise ValueError(f"{what}: rows of {tuple(key.shape[1:])} do not fit a cache of {tuple(key_cache.shape[2:])}")
    if key.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise _native.NotCovered(f"{what}: rows must be bf16, fp16 or fp32, got {key.dtype}")
    if value is not None and value.dtype != key.dtype:
        raise _native.NotCovered(f"{what}: key is {key.dtype} but value is {value.dtype}")
    blocks, page, heads, _ = key_cache.shape
    for name, rows, cache, scale in (("key", key, key_cache, k_scale), ("value", value, value_cache, v_scale)):
        if rows is None:
            continue
        if cache.dtype != torch.float8_e4m3fn:
            raise _native.NotCovered(f"{what}: {name}_cache must be float8_e4m3fn, got {cache.dtype}")
        if rows.stride(2) != 1 or cache.stride(3) != 1:
            raise _native.NotCovered(f"{what}: {name} rows and cache must have a unit stride over the head dim")
        if scale.dtype != torch.float32 or scale.dim() != 2 or scale.shape[0] < blocks or scale.shape[1] < heads:
            raise ValueError(f"{what}: the {name} scales must be fp32 [blocks >= {blocks}, heads >= {heads}], got "
                             f"{scale.dtype} {tuple(scale.shape)}")
        for t in (rows, cache, scale):
            if t.device != key.device:
                raise ValueError(f"{what}: {name} rows, cache and scales must be on one device")
    if block_table.dim() != 2 or block_table.device != key.device:
        raise ValueError(f"{what}: the block table must be [requests, blocks] on the rows' device")


def _pages_args(key, value, key_cache, value_cache, k_scale, v_scale):
    """The struct fields that writing and reading share."""
    zero = (0, 0, 0, 0)
    v, vc, vs = (zero, zero, zero) if value is None else (value.stride(), value_cache.stride(), v_scale.stride())
    kc = key_cache.stride()
    return dict(key=key.data_ptr(), value=_native.ptr(value), stride_kt=key.stride(0), stride_kh=key.stride(1), stride_vt=v[0],
                stride_vh=v[1], key_cache=key_cache.data_ptr(), value_cache=_native.ptr(value_cache), stride_kcb=kc[0],
                stride_kcs=kc[1], stride_kch=kc[2], stride_vcb=vc[0], stride_vcs=vc[1], stride_vch=vc[2],
                k_scale=k_scale.data_ptr(), v_scale=_native.ptr(v_scale), stride_ksb=k_scale.stride(0),
                stride_ksh=k_scale.stride(1), stride_vsb=vs[0], stride_vsh=vs[1], tokens=key.shape[0], heads=key.shape[1],
                dim=key.shape[2], page=key_cache.shape[1], num_blocks=key_cache.shape[0],
                dtype=_native.dtype_code(key.dtype))


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
    Positions behind a request's last row keep their bytes. Infinities saturate and do not count in ``amax``. A page
    belongs to one request. Rows whose page the table lacks, or names outside the cache, are not written.
    """
    _check_pages("write_kv_pages", key, value, key_cache, value_cache, k_scale, v_scale, block_table)
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache), ("k_scale", k_scale), ("v_scale", v_scale)):
        if t is not None and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"write_kv_pages: {name} is an expanded view: every page and head needs its own storage")
    num_reqs = query_start_loc.shape[0] - 1
    if block_table.shape[0] < num_reqs or context_lens.shape[0] < num_reqs:
        raise ValueError(f"write_kv_pages: block_table and context_lens must have {num_reqs} rows")
    if (path is None) != (path_len is None) or (path is not None and (idx_mapping is None or path.dim() != 2)):
        raise ValueError("write_kv_pages: path [slots, W], path_len [slots] and idx_mapping go together")
    if path is not None and idx_mapping.shape[0] < num_reqs:
        raise ValueError(f"write_kv_pages: idx_mapping must have {num_reqs} entries")
    for t in (context_lens, query_start_loc, path, path_len, idx_mapping):
        if t is not None and t.device != key.device:
            raise ValueError("write_kv_pages: every table must be on the rows' device")
    args = _native.WriteKvArgs(
        **_pages_args(key, value, key_cache, value_cache, k_scale, v_scale),
        block_table=_native.itab(block_table), context_lens=_native.itab(context_lens),
        query_start_loc=_native.itab(query_start_loc), idx_mapping=_native.itab(idx_mapping if path is not None else None),
        path=_native.itab(path), path_len=_native.itab(path_len), num_reqs=num_reqs, max_blocks=block_table.shape[1],
        max_rows=max_query_len, path_width=0 if path is None else path.shape[1],
        path_slots=0 if path is None else min(path.shape[0], path_len.shape[0]),
    )
    _native.launch("eagle4_write_kv_pages", args, key.device)


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
    _check_pages("read_kv_pages", key_out, value_out, key_cache, value_cache, k_scale, v_scale, block_table)
    num_reqs = start_loc.shape[0] - 1
    if block_table.shape[0] < num_reqs or start_loc.device != key_out.device:
        raise ValueError(f"read_kv_pages: block_table must have {num_reqs} rows, start_loc be on the rows' device")
    args = _native.ReadKvArgs(
        **_pages_args(key_out, value_out, key_cache, value_cache, k_scale, v_scale),
        block_table=_native.itab(block_table), start_loc=_native.itab(start_loc), num_reqs=num_reqs,
        max_blocks=block_table.shape[1], max_len=max_len,
    )
    _native.launch("eagle4_read_kv_pages", args, key_out.device)
