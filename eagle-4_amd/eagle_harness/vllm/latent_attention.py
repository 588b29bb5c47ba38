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

    Scores, sums and outputs are held in 32 bits; the softmax's weights are rounded to the rows' dtype for the second
    product, as :func:`verify_attention`'s are. The contexts decide how the work is shared out: a block table may be as wide
    as the longest model length, at no cost and with the same bits.
    """
    if q.dim() != 3 or latent_new.dim() != 2 or latent_cache.dim() != 3 or out.dim() != 3:
        raise ValueError("latent_verify_attention: q [tokens, heads, dim], latent_new [tokens, dim], latent_cache "
                         "[blocks, page, dim] and out [tokens, heads, rank]")
    (tokens, heads, dim), (blocks, page, cached), (out_tokens, out_heads, rank) = q.shape, latent_cache.shape, out.shape
    num_reqs, dtype, device = query_start_loc.shape[0] - 1, q.dtype, q.device
    if latent_new.shape != (tokens, dim) or cached != dim or out_tokens != tokens or out_heads != heads or rank >= dim:
        raise ValueError(f"latent_verify_attention: q {tuple(q.shape)}, latent_new {tuple(latent_new.shape)}, latent_cache "
                         f"{tuple(latent_cache.shape)} and out {tuple(out.shape)} do not fit")
    fp8 = latent_cache.dtype == torch.float8_e4m3fn
    if dtype not in (torch.bfloat16, torch.float16) or dtype != latent_new.dtype or dtype != out.dtype or not (
            fp8 or latent_cache.dtype == dtype):
        raise _native.NotCovered("q, latent_new and out must share a dtype (bf16 or fp16), the cache be of it or float8_e4m3fn")
    if fp8:
        if latent_scale is None:
            raise ValueError("an fp8-e4m3 cache needs latent_scale ([blocks] fp32)")
        if latent_scale.dtype != torch.float32 or latent_scale.dim() not in (1, 2) or latent_scale.shape[0] < blocks or (
                latent_scale.dim() == 2 and latent_scale.shape[1] != 1):
            raise ValueError(f"latent_scale must be fp32 [blocks >= {blocks}] or [.., 1], got {tuple(latent_scale.shape)}")
        if latent_scale.device != device:
            raise ValueError("latent_verify_attention: every tensor must be on q's device")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise _native.NotCovered("the block table must be int32 [requests, blocks] with a unit column stride")
    if masks.dtype != torch.int64 or masks.dim() != 2 or masks.stride(1) != 1:
        raise _native.NotCovered("masks must be int64 with unit row stride")
    (requests, max_blocks), (mask_rows, mask_columns) = block_table.shape, masks.shape
    if requests < num_reqs or context_lens.shape[0] < num_reqs or mask_rows < num_reqs or mask_columns < max_query_len:
        raise ValueError(f"latent_verify_attention: block_table, context_lens and masks must have {num_reqs} rows, masks "
                         f"{max_query_len} columns")
    (q_token, q_head, q_unit), (new_token, new_unit) = q.stride(), latent_new.stride()
    (cache_block, cache_slot, cache_unit), (out_token, out_head, out_unit) = latent_cache.stride(), out.stride()
    if q_unit != 1 or new_unit != 1 or cache_unit != 1 or out_unit != 1:
        raise _native.NotCovered("q, latent_new, latent_cache and out must have a unit stride over their last dim")
    for t in (latent_new, latent_cache, out, block_table, context_lens, query_start_loc, masks):
        if t.device != device:
            raise ValueError("latent_verify_attention: every tensor must be on q's device")
    itab = _native.itab
    args = _native.LatentAttnArgs(
        q.data_ptr(), q_token, q_head, latent_new.data_ptr(), new_token, latent_cache.data_ptr(), cache_block, cache_slot,
        latent_scale.data_ptr() if fp8 else 0, latent_scale.stride(0) if fp8 else 0, itab(block_table), itab(context_lens),
        itab(query_start_loc), masks.data_ptr(), masks.stride(0), out.data_ptr(), out_token, out_head, None, 0, tokens, scale,
        num_reqs, heads, rank, dim - rank, page, max_query_len, max_blocks, blocks, _native.dtype_code(dtype),
        _native.dtype_code(latent_cache.dtype))
    need = _native.library().eagle4_latent_attention_workspace(args)
    if need < 0:
        raise _native.NotCovered("eagle4_amd: latent_verify_attention does not cover this launch (shape, dtype or layout)")
    if need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)  # the torch caching allocator's
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    _native.launch("eagle4_latent_attention", args, device)
    return out
