"""Attention of decode-time draft rows whose keys are mostly shared (kernels/row_attention.py: both engines' draft
steps, sglang's draft extend), on the gfx950 kernels of ``csrc/row_attention.hip``.

Every row of a request attends to one contiguous range of the request's committed keys (found through its page
table); a draft step's rows attend, besides, to the tree nodes on their own root path:

- draft step ``step`` (``rows`` frontier rows per request): the committed keys of the window ending at the round's
  last committed position, ``[seq_len - window, seq_len - 1]``, the same for every row, plus the row's ``step``
  ancestors (KV slots, itself last);
- draft extend (``step == 0``; row ``j`` at ``seq_len + j``): the keys ``[pos - window + 1, pos]`` of its position.

One workgroup per (key split, KV head, request) reads each key once for every row of every query head of the KV
head's group; a draft step's ancestors are one more split, and a second launch merges the splits by their
log-sum-exp. Lengths are read on the device: no host planning, HIP-graph safe.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch

from eagle_harness.kernels import _native


@dataclass(frozen=True)
class RowsLaunch:
    """Launch config of :func:`rows_attention` (kernels/row_attention.py:41-51): key splits of a request's shared
    range (a draft step's tree ancestors are one more). ``block_n`` / ``num_warps`` / ``num_stages`` are the Triton
    kernel's; the gfx950 kernel keeps its own 32-key tiles and 4 waves and accepts them for the callers' sake."""

    splits: int
    block_n: int
    num_warps: int = 4
    num_stages: int = 3


STEP_WAVES = 4.0
STEP = RowsLaunch(splits=64, block_n=32, num_warps=2, num_stages=3)


def rows_padded(rows_per_request: int) -> int:
    """Rows of a request's partial block: a power of two, at least 16 (kernels/row_attention.py:60-62)."""
    return max(16, 1 << max(int(rows_per_request) - 1, 0).bit_length())


@functools.cache
def _compute_units(device: torch.device) -> int:
    """CUs of a GPU device (4 for a CPU device, where only the host-side planning runs)."""
    if device.type != "cuda":
        return 4
    return torch.cuda.get_device_properties(device).multi_processor_count


@functools.cache
def program_splits(programs: int, device: torch.device) -> int:
    """Key splits per (request, head) program: the power of two that gives every CU at least one program."""
    return 1 << max(0, math.ceil(math.log2(max(1, -(-_compute_units(device) // max(1, programs))))))


def step_splits(programs: int, device: torch.device) -> int:
    """Key splits of a draft step launched as ``programs`` (request, head) programs per split
    (kernels/row_attention.py:229-233): the split count is a power of two, chosen so that splits x programs comes
    closest to STEP_WAVES programs per CU when compared on a log2 scale."""
    waves_wanted = STEP_WAVES * _compute_units(device) / programs
    exponent = round(math.log2(waves_wanted))
    return 2 ** exponent if exponent > 0 else 1


def _cache_strides(cache: torch.Tensor) -> tuple[int, int, int]:
    """Element strides (per page, per slot within its page, per KV head) of a cache view. A ``[pages, page, heads,
    D]`` view has all three; a ``[slots, heads, D]`` view is read as pages of one slot, so its slot stride is 0."""
    if cache.dim() == 4:
        per_page, per_slot, per_head = cache.stride(0), cache.stride(1), cache.stride(2)
    else:
        per_page, per_slot, per_head = cache.stride(0), 0, cache.stride(1)
    return per_page, per_slot, per_head


def _check_fp8(q, keys, values, out, k_scale, v_scale) -> None:
    if keys.dtype != torch.float8_e4m3fn or values is None or values.dtype != torch.float8_e4m3fn:
        raise _native.NotCovered("caches with scales must be float8_e4m3fn keys and values")
    if q.dtype not in (torch.bfloat16, torch.float16) or out.dtype != q.dtype:
        raise _native.NotCovered("q and out over fp8 pages must share one 16-bit dtype")
    if values.shape != keys.shape:
        raise ValueError(f"values {tuple(values.shape)} are not shaped as keys {tuple(keys.shape)}")
    pages, heads = keys.shape[0], keys.shape[-2]
    for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
        if scale.dtype != torch.float32 or scale.dim() != 2 or scale.shape[0] < pages or scale.shape[1] < heads:
            raise ValueError(f"{name} must be fp32 [pages >= {pages}, kv_heads >= {heads}], got {scale.dtype} {tuple(scale.shape)}")
        if scale.device != q.device:
            raise ValueError(f"{name} must be on {q.device}")


def rows_attention(
    q: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor | None,
    out: torch.Tensor,
    part_out: torch.Tensor,
    part_lse: torch.Tensor,
    table: torch.Tensor,
    seq_lens: torch.Tensor,
    ancestors: torch.Tensor | None,
    *,
    rows_per_request: int,
    step: int,
    window: int,
    scale: float,
    launch: RowsLaunch,
    table_rows: torch.Tensor | None = None,
    table_page: int = 1,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> None:
    """Attention of ``q`` ``[bs * rows_per_request, heads, D]`` into ``out`` (same shape).

    ``step == 0``: extend rows (row ``j`` of request ``b`` at ``seq_lens[b] + j``, causal); else the rows of draft
    step ``step`` over the committed window plus ``ancestors[b, row, :step]`` (KV slots). ``keys`` / ``values``:
    the layer's KV cache as ``[slots, kv_heads, D]`` or ``[pages, page, kv_heads, D]`` views; for a packed cache
    pass ``keys`` with last dimension ``2 * D`` and ``values=None``. Consecutive groups of ``heads // kv_heads`` query
    heads share one KV head. The key at position ``p`` of request ``b`` is slot
    ``table[table_rows[b], p // table_page] * table_page + p % table_page`` (row ``b`` without ``table_rows``).
    ``part_out`` / ``part_lse``: scratch of at least ``bs * heads * (launch.splits + 1) *
    rows_padded(rows_per_request)`` rows (kernels/row_attention.py:251-328).

    Beyond the reference: ``float8_e4m3fn`` caches (``keys`` and ``values``, as ``write_kv_pages`` fills them) with
    ``k_scale`` / ``v_scale`` fp32 ``[pages, kv_heads]`` (any strides), under bf16 or fp16 rows. Value scales below 2^-100 count
    as 0. A row that sees no key gives zeros.
    """
    rows, heads, head_dim = q.shape
    kv_heads = keys.shape[-2]
    if kv_heads <= 0 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be divisible by KV heads ({kv_heads})")
    if step > 0 and ancestors is None:
        raise ValueError("a draft step needs its rows' ancestors")
    if (k_scale is None) != (v_scale is None):
        raise ValueError("k_scale and v_scale go together")
    if k_scale is not None:
        _check_fp8(q, keys, values, out, k_scale, v_scale)
    elif q.dtype != keys.dtype or out.dtype != q.dtype or (values is not None and values.dtype != q.dtype):
        raise _native.NotCovered("q, the caches and out must share one 16-bit dtype")
    for name, t in (("q", q), ("out", out), ("keys", keys)) + ((("values", values),) if values is not None else ()):
        if t.stride(-1) != 1:
            raise _native.NotCovered(f"{name} must have a unit stride over the head dim")
    if part_out.dtype != torch.float32 or part_lse.dtype != torch.float32 or not part_out.is_contiguous():
        raise _native.NotCovered("the partials are contiguous fp32 scratch")
    if table.dtype != torch.int32 or table.stride(-1) != 1:
        raise _native.NotCovered("the page table must be int32 with unit stride")
    bs = rows // rows_per_request
    kst = _cache_strides(keys)
    vst = _cache_strides(values) if values is not None else kst
    anc = None
    if step > 0:
        anc = ancestors if ancestors.dtype == torch.int32 and ancestors.is_contiguous() else ancestors.to(
            torch.int32).contiguous()
    args = _native.RowAttnArgs(
        q=q.data_ptr(),
        stride_q_row=q.stride(0),
        stride_q_head=q.stride(1),
        keys=keys.data_ptr(),
        values=_native.ptr(values),
        k_stride_page=kst[0],
        k_stride_slot=kst[1],
        k_stride_head=kst[2],
        v_stride_page=vst[0],
        v_stride_slot=vst[1],
        v_stride_head=vst[2],
        out=out.data_ptr(),
        stride_o_row=out.stride(0),
        stride_o_head=out.stride(1),
        part_out=part_out.data_ptr(),
        part_lse=part_lse.data_ptr(),
        part_rows=min(part_out.shape[0], part_lse.numel()),
        table=table.data_ptr(),
        stride_table=table.stride(0),
        table_rows=_native.itab(table_rows),
        seq_lens=_native.itab(seq_lens),
        ancestors=_native.ptr(anc),
        max_depth=anc.shape[-1] if anc is not None else 1,
        table_page=table_page,
        cache_page=1 if keys.dim() == 3 else keys.shape[1],
        bs=bs,
        rows_per_request=rows_per_request,
        rows_padded=rows_padded(rows_per_request),
        heads=heads,
        kv_heads=kv_heads,
        head_dim=head_dim,
        dtype=_native.dtype_code(q.dtype),
        step=step,
        window=window,
        splits=launch.splits,
        scale=scale,
    )
    if k_scale is None:
        _native.launch("eagle4_row_attention", args, q.device)
        return
    if table.dim() != 2 or 0 in table.shape or keys.shape[0] == 0:
        raise ValueError("the page table must be [requests, entries], and the caches hold pages")
    fp8 = _native.RowAttnFp8Args(args, k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), v_scale.stride(0),
                                 v_scale.stride(1), table.shape[0], table.shape[1], keys.shape[0])
    _native.launch("eagle4_row_attention_fp8", fp8, q.device)
