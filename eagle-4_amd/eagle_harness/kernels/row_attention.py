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
_MOST = (1 << 31) - 1  # of a 32-bit field; a longer window is the whole context
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


def _cache_strides(stride: tuple) -> tuple[int, int, int]:
    """Element strides (per page, per slot within its page, per KV head) of a cache view, of its own. A ``[pages, page,
    heads, D]`` view has all three; a ``[slots, heads, D]`` view is read as pages of one slot, so its slot stride is 0."""
    if len(stride) == 4:
        return stride[0], stride[1], stride[2]
    return stride[0], 0, stride[1]


def _check_fp8(q, keys, values, out, k_scale, v_scale, part_out, part_lse, table, seq_lens, ancestors, table_rows, rows_per_request,
               step) -> None:
    fp8, dtype, rows_shape, shape = torch.float8_e4m3fn, q.dtype, q.shape, keys.shape
    if values is None or keys.dtype != fp8 or values.dtype != fp8:
        raise _native.NotCovered("caches with scales must be float8_e4m3fn keys and values")
    if (dtype != torch.bfloat16 and dtype != torch.float16) or out.dtype != dtype:
        raise _native.NotCovered("q and out over fp8 pages must share one 16-bit dtype")
    if values.shape != shape or not 3 <= len(shape) <= 4 or shape[-1] != rows_shape[2] or shape[0] == 0:
        raise ValueError(f"keys {tuple(shape)} and values {tuple(values.shape)} must be alike, [pages, page, kv_heads, {rows_shape[2]}]")
    if out.shape != rows_shape:
        raise ValueError(f"out must be {tuple(rows_shape)}, got {tuple(out.shape)}")
    pages, heads = shape[0], shape[-2]
    for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
        have = scale.shape
        if scale.dtype != torch.float32 or len(have) != 2 or have[0] < pages or have[1] < heads:
            raise ValueError(f"{name} must be fp32 [pages >= {pages}, kv_heads >= {heads}], got {scale.dtype} {tuple(have)}")
    if part_out.dim() != 2 or part_out.shape[1] != rows_shape[2] or not part_lse.is_contiguous():
        raise ValueError(f"part_out must be [rows, {rows_shape[2]}], part_lse contiguous, got {tuple(part_out.shape)}")
    if rows_per_request < 1 or rows_shape[0] % rows_per_request:
        raise ValueError(f"{rows_shape[0]} rows are not {rows_per_request} a request")
    bs = rows_shape[0] // rows_per_request
    if table.dim() != 2 or seq_lens.dim() == 0 or (bs > 0 and table.numel() == 0) or seq_lens.shape[0] < bs \
            or (table_rows is not None and table_rows.dim() == 0) or (table if table_rows is None else table_rows).shape[0] < bs:
        raise ValueError(f"the page table must be [requests, entries], seq_lens and table_rows [{bs}]")
    if step > 0 and (ancestors.shape[-1] < step or ancestors.numel() < bs * rows_per_request * ancestors.shape[-1]):
        raise ValueError(f"ancestors must be [{bs}, {rows_per_request}, >= {step}], got {tuple(ancestors.shape)}")
    where = q.get_device()
    for t in (keys, values, out, k_scale, v_scale, part_out, part_lse, table, seq_lens, ancestors if step > 0 else None, table_rows):
        if t is not None and t.get_device() != where:
            raise ValueError(f"every tensor must be on the rows' device, {q.device}, got {t.device}")


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
    ``k_scale`` / ``v_scale`` fp32 ``[pages, kv_heads]`` (any strides; not negative), under bf16 or fp16 rows. Value scales below
    2^-100 count as 0. Softmax weights enter the product with the values in bf16 under bf16 rows (sums and the denominator are in
    32 bits), in 16 bits over the range of 32-bit floats under fp16 rows. Keys end with the page table (a row behind it sees those before),
    and nothing is read past the cache's last page. A row that sees no key gives zeros.
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
        _check_fp8(q, keys, values, out, k_scale, v_scale, part_out, part_lse, table, seq_lens, ancestors, table_rows,
                   rows_per_request, step)
    elif q.dtype != keys.dtype or out.dtype != q.dtype or (values is not None and values.dtype != q.dtype):
        raise _native.NotCovered("q, the caches and out must share one 16-bit dtype")
    q_stride, out_stride, k_stride = q.stride(), out.stride(), keys.stride()
    v_stride = k_stride if values is None else values.stride()
    if q_stride[-1] != 1 or out_stride[-1] != 1 or k_stride[-1] != 1 or v_stride[-1] != 1:
        strides = {"q": q_stride, "out": out_stride, "keys": k_stride, "values": v_stride}
        name = next(n for n, stride in strides.items() if stride[-1] != 1)
        raise _native.NotCovered(f"{name} must have a unit stride over the head dim")
    if part_out.dtype != torch.float32 or part_lse.dtype != torch.float32 or not part_out.is_contiguous():
        raise _native.NotCovered("the partials are contiguous fp32 scratch")
    table_stride = table.stride()
    if table.dtype != torch.int32 or table_stride[-1] != 1:
        raise _native.NotCovered("the page table must be int32 with unit stride")
    if abs(table_page) > _MOST:
        raise ValueError(f"table_page must be at most {_MOST}, got {table_page}")
    bs = rows // rows_per_request
    kst, vst = _cache_strides(k_stride), _cache_strides(v_stride)
    anc = None
    if step > 0:
        anc = ancestors if ancestors.dtype == torch.int32 and ancestors.is_contiguous() else ancestors.to(
            torch.int32).contiguous()
    args = _native.RowAttnArgs(  # by position, as the struct has them: by name it costs more than the rest of the call
        q.data_ptr(), q_stride[0], q_stride[1], keys.data_ptr(), _native.ptr(values), kst[0], kst[1], kst[2], vst[0], vst[1], vst[2],
        out.data_ptr(), out_stride[0], out_stride[1], part_out.data_ptr(), part_lse.data_ptr(),
        min(part_out.shape[0], part_lse.numel()), table.data_ptr(), table_stride[0], _native.itab(table_rows),
        _native.itab(seq_lens), _native.ptr(anc), anc.shape[-1] if anc is not None else 1, table_page,
        1 if len(k_stride) == 3 else keys.shape[1], bs, rows_per_request, rows_padded(rows_per_request), heads, kv_heads, head_dim,
        _native.dtype_code(q.dtype), step, min(window, _MOST), launch.splits, scale)
    if k_scale is None:
        _native.launch("eagle4_row_attention", args, q.device)
        return
    ks, vs, (height, width) = k_scale.stride(), v_scale.stride(), table.shape
    fp8 = _native.RowAttnFp8Args(args, k_scale.data_ptr(), v_scale.data_ptr(), ks[0], ks[1], vs[0], vs[1], height, width, keys.shape[0])
    _native.launch("eagle4_row_attention_fp8", fp8, q.device)
