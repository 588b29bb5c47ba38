"""Tree-verify attention of layers whose keys and values are one latent row a token (``csrc/latent_attention.hip``).

A token's cached row holds ``rank`` latent values and ``rope`` rotary ones, shared by all heads: the row is every head's key
and its first ``rank`` values every head's value. In this (absorbed) form ``q`` holds each head's query already taken
through the key half of the up-projection, and the caller takes ``out`` through the value half. It is
:func:`verify_attention`'s counterpart: the same page tables, context lengths and ancestor masks, one query row a request
(a decode step) to 64.
"""

from __future__ import annotations

from typing import Optional

import torch

from eagle_harness.kernels import _native


def latent_verify_attention(
    q: torch.Tensor,
    latent_new: torch.Tensor,
    latent_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    masks: torch.Tensor,
    scale: float,
    out: torch.Tensor,
    *,
    max_query_len: int,
    latent_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Latent verify attention into ``out`` ``[tokens, heads, rank]`` (rows past the last request's are left alone).

    ``q`` ``[tokens, heads, rank + rope]``; ``latent_new`` ``[tokens, rank + rope]`` the new tokens' rows; ``latent_cache``
    ``[blocks, page, rank + rope]`` holds each request's first ``context_lens[b]`` tokens through ``block_table[b]``;
    ``masks[b, r]`` has bit ``j`` set iff new token ``j`` is row ``r`` or one of its ancestors. Every request has at most
    ``max_query_len`` (<= 64) rows. bf16 or fp16, the cache of the rows' dtype or fp8-e4m3 with ``latent_scale``, one fp32
    scale a page (``[blocks]``, or ``[blocks, 1]`` as :func:`~eagle_harness.vllm.kv_pages.write_kv_pages` keeps it). rank 256 or
    512, rope 64. A row that sees no key gives zeros; a position whose page id lies outside the cache is not seen.
    """
    if q.dim() != 3 or latent_new.dim() != 2 or latent_cache.dim() != 3 or out.dim() != 3:
        raise ValueError("latent_verify_attention: q [tokens, heads, dim], latent_new [tokens, dim], latent_cache "
                         "[blocks, page, dim] and out [tokens, heads, rank]")
    tokens, heads, dim = q.shape
    blocks, page, _ = latent_cache.shape
    rank, num_reqs = out.shape[2], query_start_loc.shape[0] - 1
    if latent_new.shape != (tokens, dim) or latent_cache.shape[2] != dim or out.shape[:2] != (tokens, heads) or rank >= dim:
        raise ValueError(f"latent_verify_attention: q {tuple(q.shape)}, latent_new {tuple(latent_new.shape)}, latent_cache "
                         f"{tuple(latent_cache.shape)} and out {tuple(out.shape)} do not fit")
    fp8 = latent_cache.dtype == torch.float8_e4m3fn
    if q.dtype not in (torch.bfloat16, torch.float16) or q.dtype != latent_new.dtype or q.dtype != out.dtype or not (
            fp8 or latent_cache.dtype == q.dtype):
        raise _native.NotCovered("q, latent_new and out must share a dtype (bf16 or fp16), the cache be of it or float8_e4m3fn")
    if fp8:
        if latent_scale is None:
            raise ValueError("an fp8-e4m3 cache needs latent_scale ([blocks] fp32)")
        if latent_scale.dtype != torch.float32 or latent_scale.dim() not in (1, 2) or latent_scale.shape[0] < blocks or (
                latent_scale.dim() == 2 and latent_scale.shape[1] < 1):
            raise ValueError(f"latent_scale must be fp32 [blocks >= {blocks}], got {tuple(latent_scale.shape)}")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise _native.NotCovered("the block table must be int32 [requests, blocks] with a unit column stride")
    if masks.dtype != torch.int64 or masks.dim() != 2 or masks.stride(1) != 1:
        raise _native.NotCovered("masks must be int64 with unit row stride")
    if (block_table.shape[0] < num_reqs or context_lens.shape[0] < num_reqs or masks.shape[0] < num_reqs
            or masks.shape[1] < max_query_len):
        raise ValueError(f"latent_verify_attention: block_table, context_lens and masks must have {num_reqs} rows, masks "
                         f"{max_query_len} columns")
    for name, t in (("q", q), ("latent_new", latent_new), ("latent_cache", latent_cache), ("out", out)):
        if t.stride(-1) != 1:
            raise _native.NotCovered(f"{name} must have a unit stride over its last dim")
    for t in (latent_new, latent_cache, out, block_table, context_lens, query_start_loc, masks, latent_scale if fp8 else None):
        if t is not None and t.device != q.device:
            raise ValueError("latent_verify_attention: every tensor must be on q's device")
    args = _native.LatentAttnArgs(
        q=q.data_ptr(), stride_qt=q.stride(0), stride_qh=q.stride(1), latent_new=latent_new.data_ptr(),
        stride_nt=latent_new.stride(0), cache=latent_cache.data_ptr(), stride_cb=latent_cache.stride(0),
        stride_cs=latent_cache.stride(1), scale_page=latent_scale.data_ptr() if fp8 else 0,
        stride_sp=latent_scale.stride(0) if fp8 else 0, block_table=_native.itab(block_table),
        context_lens=_native.itab(context_lens), query_start_loc=_native.itab(query_start_loc), masks=masks.data_ptr(),
        stride_mask=masks.stride(0), out=out.data_ptr(), stride_ot=out.stride(0), stride_oh=out.stride(1), tokens=tokens,
        scale=scale, num_reqs=num_reqs, heads=heads, rank=rank, rope=dim - rank, page=page, max_query_len=max_query_len,
        max_blocks=block_table.shape[1], num_blocks=blocks, dtype=_native.dtype_code(q.dtype),
        cache_dtype=_native.dtype_code(latent_cache.dtype),
    )
    need = _native.library().eagle4_latent_attention_workspace(args)
    if need < 0:
        raise _native.NotCovered("eagle4_amd: latent_verify_attention does not cover this launch (shape, dtype or layout)")
    if need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)  # the torch caching allocator's
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    _native.launch("eagle4_latent_attention", args, q.device)
    return out
