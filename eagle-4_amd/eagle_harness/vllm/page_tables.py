"""Block tables that follow the requests' lengths, and the cache slots of a batch's rows (``csrc/page_tables.hip``).

Tables, page counts and the stack of free pages stay on the GPU, indexed by request state slot as
:class:`~eagle_harness.vllm.verify_layout.TreeStore` is: :func:`resize_tables` takes and gives pages for the lengths that a round needs,
:func:`slot_maps` gives the batch its block table (what the attentions and the page writes take) and each of its rows its
place in the cache (what draft steps keep as ``ancestors``). Both can be captured in a graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from eagle_harness.kernels import _native


def _tables(what: str, block_table: torch.Tensor, num_pages: torch.Tensor, idx_mapping: torch.Tensor, page: int) -> tuple:
    """Checks what both operators share: (slots, max_pages, row stride, requests, the device's number)."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or num_pages.dtype != torch.int32:
        raise ValueError(f"{what}: block_table [slots, pages] and num_pages [slots] must be int32")
    (slots, most), (stride, column), where = block_table.shape, block_table.stride(), block_table.get_device()
    if slots < 1 or most < 1:
        raise ValueError(f"{what}: block_table is empty")
    if (column != 1 and most != 1) or (stride < most and slots > 1):
        raise _native.NotCovered(f"{what}: block_table must have a unit column stride and rows of their own storage")
    if num_pages.shape != (slots,) or not num_pages.is_contiguous():
        raise ValueError(f"{what}: num_pages must be contiguous, one entry for each of the {slots} slots")
    if idx_mapping.dim() != 1 or not 0 < page < 1 << 31:
        raise ValueError(f"{what}: idx_mapping must be a vector and page from 1 to 2^31 - 1")
    if num_pages.get_device() != where or idx_mapping.get_device() != where:
        raise ValueError(f"{what}: every tensor must be on {block_table.device}")
    return slots, most, stride, idx_mapping.shape[0], where


def resize_tables(
    block_table: torch.Tensor,
    num_pages: torch.Tensor,
    idx_mapping: torch.Tensor,
    lens: torch.Tensor,
    free_pages: torch.Tensor,
    num_free: torch.Tensor,
    page: int,
) -> None:
    """Brings every request of the batch to the pages that its length needs, in place.

    ``block_table`` [slots, pages] and ``num_pages`` [slots] int32: the pages that each state slot holds; ``idx_mapping``
    [requests] the slots of the batch (each at most once, or its pages are given back or taken twice; a negative one is a
    padded request), ``lens`` [requests] their lengths
    (int32 / int64), context and the rows to come. ``free_pages`` int32, as long as there are pages, with ``num_free`` [1]
    int32: a stack of the free ones.

    First every request that holds more than ``ceil(len / page)`` pages gives the rest back, the last request's last page
    first; then the others take from the stack's top, in the batch's order, each page in turn. Where the free pages do not
    suffice, the requests from the first one on whose pages, with those before it, are not there keep what they hold: a
    request got its pages iff ``num_pages[slot] * page >= len``. A length that the table has no room for changes nothing
    of its request. Giving back in the same order what was just taken leaves the stack as it was. Table entries behind a
    request's pages are not cleared. Nothing happens at all if ``num_free`` and what comes back are more than ``free_pages`` holds.
    """
    slots, most, stride, requests, where = _tables("resize_tables", block_table, num_pages, idx_mapping, page)
    if lens.dim() != 1 or lens.shape[0] < requests:
        raise ValueError(f"resize_tables: lens must be [{requests}]")
    if free_pages.dtype != torch.int32 or free_pages.dim() != 1 or not free_pages.is_contiguous():
        raise ValueError("resize_tables: free_pages must be a contiguous int32 vector")
    if num_free.dtype != torch.int32 or num_free.numel() != 1:
        raise ValueError("resize_tables: num_free must be one int32")
    if lens.get_device() != where or free_pages.get_device() != where or num_free.get_device() != where:
        raise ValueError(f"resize_tables: every tensor must be on {block_table.device}")
    if requests == 0:
        return
    args = _native.ResizeTablesArgs(block_table.data_ptr(), stride, num_pages.data_ptr(), _native.itab(idx_mapping),
                                    _native.itab(lens), free_pages.data_ptr(), num_free.data_ptr(), free_pages.shape[0], requests,
                                    slots, most, page)
    _native.launch("eagle4_resize_tables", args, block_table.device)


def slot_maps(
    block_table: torch.Tensor,
    num_pages: torch.Tensor,
    idx_mapping: torch.Tensor,
    context_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    page: int,
    *,
    slots: torch.Tensor,
    batch_table: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The cache slot of every row of a batch, and the batch's own block table, into given buffers: ``(slots, batch_table)``.

    Row ``j`` of request ``r`` (rows ``query_start_loc[r] ..``) is position ``context_lens[r] + j`` of state slot ``idx_mapping[r]``;
    ``slots`` (contiguous int64, as long as the batch is padded to) gets ``block_table[slot, position // page] * page + position %
    page``, -1 where the request holds no such page, and -1 before the first and behind the last request's rows. ``batch_table`` [requests, pages] int32
    gets each request's pages and 0 behind them; request rows behind the batch are left as they were.
    """
    state_slots, most, stride, requests, where = _tables("slot_maps", block_table, num_pages, idx_mapping, page)
    if query_start_loc.dim() != 1 or context_lens.dim() != 1 or query_start_loc.shape[0] < requests + 1 or context_lens.shape[0] < requests:
        raise ValueError(f"slot_maps: query_start_loc must be [{requests + 1}] and context_lens [{requests}]")
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slot_maps: slots must be a contiguous int64 vector")
    batch_stride = 0
    if batch_table is not None:
        if batch_table.dtype != torch.int32 or batch_table.dim() != 2 or batch_table.shape[0] < requests or batch_table.shape[1] != most:
            raise ValueError(f"slot_maps: batch_table must be int32 [{requests}, {most}]")
        batch_stride, column = batch_table.stride()
        if (column != 1 and most != 1) or (batch_stride < most and requests > 1):
            raise _native.NotCovered("slot_maps: batch_table must have a unit column stride and rows of their own storage")
        if batch_table.get_device() != where:
            raise ValueError(f"slot_maps: every tensor must be on {block_table.device}")
        at, to = block_table.data_ptr(), batch_table.data_ptr()
        if requests and at < to + 4 * ((requests - 1) * batch_stride + most) and to < at + 4 * ((state_slots - 1) * stride + most):
            if not _native.apart(at, ((state_slots, 4 * stride),), 4 * most, to, ((requests, 4 * batch_stride),), 4 * most):
                raise ValueError("slot_maps: batch_table must not overlap block_table")
    if context_lens.get_device() != where or query_start_loc.get_device() != where or slots.get_device() != where:
        raise ValueError(f"slot_maps: every tensor must be on {block_table.device}")
    if requests == 0 and slots.shape[0] == 0:
        return slots, batch_table
    args = _native.SlotMapsArgs(block_table.data_ptr(), stride, num_pages.data_ptr(), _native.itab(idx_mapping),
                                _native.itab(context_lens), _native.itab(query_start_loc), slots.data_ptr(),
                                _native.ptr(batch_table), batch_stride, slots.shape[0], requests, state_slots, most, page)
    _native.launch("eagle4_slot_maps", args, block_table.device)
    return slots, batch_table
