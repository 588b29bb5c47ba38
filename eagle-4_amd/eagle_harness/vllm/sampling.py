"""Rows of logits under temperature, top-k, top-p and min-p (``csrc/sample_rows.hip``): a draft's tokens drawn from given uniform
numbers, with the distribution that :func:`~eagle_harness.vllm.tree_accept.sample_tree` takes as ``draft_probs``, and a
target's rows cut to what the rules keep, for that walk.

A row's weights are ``w = exp((logits - max) / temperature)``, its order is descending in the logits, the lower index first
among equals. Each rule keeps a beginning of the order, in this sequence:

- ``min_p``: the tokens with ``w >= min_p`` (0: all);
- ``top_k``: the first ``top_k`` tokens (0, or from the vocabulary's size on: all);
- ``top_p``: of what these two leave, with mass ``Z1``, the tokens with less than ``top_p Z1`` before them (from 1 on: all).

The first token is always kept. A temperature that is not above 0, or a row whose maximum is not finite, leaves the argmax alone
(the first index; NaN is the largest value). Weights are computed in 64 bits, their sums are exact.
"""

from __future__ import annotations

from typing import Optional

import torch

from eagle_harness.kernels import _native

_DTYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32}
PROBS, LOGITS = 1, 2
MAX_VOCAB, MAX_DRAWS = 1 << 18, 64


def _rows_args(what: str, logits: torch.Tensor, temperature: torch.Tensor, top_k: Optional[torch.Tensor],
               top_p: Optional[torch.Tensor], min_p: Optional[torch.Tensor], entries: Optional[torch.Tensor]) -> tuple:
    """Checks what both operators share: the dtype's code and the struct's first fields."""
    if logits.dim() != 2:
        raise ValueError(f"{what}: logits must be [rows, vocab], got {tuple(logits.shape)}")
    (rows, vocab), (stride, column) = logits.shape, logits.stride()
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise _native.NotCovered(f"{what}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if (column != 1 and vocab != 1) or not 0 < vocab <= MAX_VOCAB:
        raise _native.NotCovered(f"{what}: logits must have a unit column stride and 1 to {MAX_VOCAB} columns")
    device, count = logits.device, temperature.shape[0] if temperature.dim() == 1 else -1
    for name, t, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is None:
            continue
        if t.dtype != dtype or t.shape != (count,) or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{what}: {name} must be a contiguous {dtype} vector as long as temperature, on {device}")
    if entries is None:
        if count < rows:
            raise ValueError(f"{what}: {rows} rows need as many temperatures, or entries that name theirs")
    elif entries.dim() != 1 or entries.shape[0] < rows or entries.device != device:
        raise ValueError(f"{what}: entries must be [{rows}] on {device}")
    if count < 1 and rows > 0:
        raise ValueError(f"{what}: no temperature is given")
    return code, (logits.data_ptr(), stride, _native.itab(entries), temperature.data_ptr(), _native.ptr(top_k),
                  _native.ptr(top_p), _native.ptr(min_p))


def _out_stride(what: str, name: str, out: torch.Tensor, logits: torch.Tensor) -> int:
    """The row stride of a given output of the logits' shape."""
    if out.shape != logits.shape or out.device != logits.device:
        raise ValueError(f"{what}: {name} must have the logits' shape and device")
    (rows, vocab), (stride, column) = out.shape, out.stride()
    if (column != 1 and vocab != 1) or (rows > 1 and stride < vocab):
        raise _native.NotCovered(f"{what}: {name} must have a unit column stride and rows of their own storage")
    return stride


def _overlap(logits: torch.Tensor, out: torch.Tensor, out_stride: int) -> bool:
    (rows, vocab), a, b, size, out_size = logits.shape, logits.data_ptr(), out.data_ptr(), logits.element_size(), out.element_size()
    stride = logits.stride(0)
    if rows == 0 or a >= b + out_size * ((rows - 1) * out_stride + vocab) or b >= a + size * ((rows - 1) * stride + vocab):
        return False
    return not _native.apart(a, ((rows, size * stride),), size * vocab, b, ((rows, out_size * out_stride),), out_size * vocab)


def draw_tokens(
    logits: torch.Tensor,
    coins: torch.Tensor,
    temperature: torch.Tensor,
    top_k: Optional[torch.Tensor] = None,
    top_p: Optional[torch.Tensor] = None,
    min_p: Optional[torch.Tensor] = None,
    *,
    entries: Optional[torch.Tensor] = None,
    probs: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Tokens drawn from each row's kept part, int64 of ``coins``' shape.

    ``logits`` [rows, vocab] (bf16 / fp16 / fp32, unit column stride); ``coins`` [rows] or [rows, draws] (at most 64) fp32
    uniform numbers in [0, 1), contiguous: each draws one token of its row, independently. ``temperature``, ``top_k``
    (int32), ``top_p`` and ``min_p`` (fp32; None: off) are vectors over requests, ``entries`` [rows] (int32 / int64) the
    request of each row; without it row ``n`` takes entry ``n``. A row whose entry is negative or past the vectors (a
    padded one) gets tokens of 0, which a captured step may look up; its row of ``probs`` is left as it was.

    With ``Z`` the mass kept, the token is the first of the order whose running mass exceeds ``coin * Z``. ``probs`` [rows,
    vocab] (bf16 / fp16 / fp32, no element shared with the logits) is filled with ``w / Z`` on the kept tokens, 0 elsewhere.
    """
    code, fields = _rows_args("draw_tokens", logits, temperature, top_k, top_p, min_p, entries)
    rows, vocab = logits.shape
    draws = 1 if coins.dim() == 1 else coins.shape[1] if coins.dim() == 2 else 0
    if not 0 < draws <= MAX_DRAWS:
        raise ValueError(f"draw_tokens: coins must be [rows] or [rows, 1 to {MAX_DRAWS}], got {tuple(coins.shape)}")
    if coins.dtype != torch.float32 or coins.shape[0] != rows or not coins.is_contiguous() or coins.device != logits.device:
        raise ValueError(f"draw_tokens: coins must be contiguous fp32 for {rows} rows on {logits.device}")
    out, stride, kind, out_code = None, 0, 0, 0
    if probs is not None:
        out, stride, kind, out_code = probs.data_ptr(), _out_stride("draw_tokens", "probs", probs, logits), PROBS, _DTYPES.get(probs.dtype)
        if out_code is None:
            raise _native.NotCovered(f"draw_tokens: probs must be bf16, fp16 or fp32, got {probs.dtype}")
        if _overlap(logits, probs, stride):
            raise ValueError("draw_tokens: probs must not overlap the logits")
    tokens = torch.empty(coins.shape, dtype=torch.int64, device=logits.device)
    if rows == 0:
        return tokens
    args = _native.SampleRowsArgs(*fields, coins.data_ptr(), tokens.data_ptr(), out, stride, rows, temperature.shape[0], vocab,
                                  draws, code, kind, out_code, 0)
    _native.launch("eagle4_sample_rows", args, logits.device)
    return tokens


def truncate_logits(
    logits: torch.Tensor,
    temperature: torch.Tensor,
    top_k: Optional[torch.Tensor] = None,
    top_p: Optional[torch.Tensor] = None,
    min_p: Optional[torch.Tensor] = None,
    *,
    entries: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``logits`` with -inf for every token outside its row's kept part: what a target that samples under these rules gives
    :func:`~eagle_harness.vllm.tree_accept.sample_tree`, with the same temperatures.

    Arguments as :func:`draw_tokens`'. ``out`` [rows, vocab] of the logits' dtype takes the rows (``out=logits``: in place;
    any other overlap is not allowed); None: a new tensor. Rows of entries outside the vectors keep their logits: they are not written in a
    given ``out``, and copied into a new tensor."""
    code, fields = _rows_args("truncate_logits", logits, temperature, top_k, top_p, min_p, entries)
    rows, vocab = logits.shape
    copy_padded = out is None
    if copy_padded:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        stride = vocab
    else:
        stride = _out_stride("truncate_logits", "out", out, logits)
        if out.dtype != logits.dtype:
            raise ValueError(f"truncate_logits: out must be {logits.dtype}, got {out.dtype}")
        if (out.data_ptr() != logits.data_ptr() or (rows > 1 and stride != logits.stride(0))) and _overlap(logits, out, stride):
            raise ValueError("truncate_logits: out may be the logits themselves, but not overlap them otherwise")
    if rows == 0:
        return out
    args = _native.SampleRowsArgs(*fields, None, None, out.data_ptr(), stride, rows, temperature.shape[0], vocab, 0, code, LOGITS,
                                  code, copy_padded)
    _native.launch("eagle4_sample_rows", args, logits.device)
    return out
