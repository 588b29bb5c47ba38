"""Rotary positions of queries and keys (``csrc/rotary.hip``), before :func:`~eagle_harness.vllm.verify_attention.verify_attention`,
``rows_attention`` or a page write: a tree's rows at the positions that :func:`~eagle_harness.vllm.verify_layout.stage_tree` leaves.

The angles come from 64-bit frequencies, ``position * frequency`` in 64 bits: there is no table of cosines whose length bounds the
context, and far positions keep their angle. :func:`rotary_frequencies` makes the frequencies, plain or scaled for long contexts.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from eagle_harness.kernels import _native

_DTYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32}


def rotary_frequencies(
    dim: int,
    base: float = 10000.0,
    *,
    scaling: str = "none",
    stretch: float = 1.0,
    trained: int = 0,
    fast: float = 32.0,
    slow: float = 1.0,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """``(frequencies [dim / 2] fp64 in radians a position, factor)`` for :func:`rotate_rows`: ``base ** (-2 i / dim)`` for the pair
    ``i`` of the ``dim`` turned elements, for contexts of ``stretch`` times the trained length by

    - ``"none"``: as trained;
    - ``"linear"``: every frequency divided by ``stretch``;
    - ``"ntk"``: the base times ``stretch ** (dim / (dim - 2))``, which leaves the fastest pair and divides the slowest by
      ``stretch``;
    - ``"yarn"``: pairs that turn at least ``fast`` times within the ``trained`` positions stay, those that turn at most ``slow``
      times are divided by ``stretch``, evenly over the pair's number in between; ``factor`` is ``0.1 ln(stretch) + 1``.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even and positive, got {dim}")
    if not base > 1.0 or not stretch >= 1.0:
        raise ValueError(f"rotary_frequencies: base must be above 1 and stretch at least 1, got {base}, {stretch}")
    half, factor = dim // 2, 1.0
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("rotary_frequencies: 'ntk' needs at least two pairs")
        base = base * stretch ** (dim / (dim - 2))
    pair = torch.arange(half, dtype=torch.float64)
    frequencies = torch.pow(torch.tensor(base, dtype=torch.float64), -pair / half)
    if scaling == "linear":
        frequencies = frequencies / stretch
    elif scaling == "yarn":
        if trained < 1 or not fast > slow > 0:
            raise ValueError("rotary_frequencies: 'yarn' needs the trained length, and fast > slow > 0")
        # the pair that turns so many times within the trained positions
        place = lambda turns: half * math.log(trained / (turns * 2 * math.pi)) / math.log(base)  # noqa: E731
        low, high = max(math.floor(place(fast)), 0), min(math.ceil(place(slow)), dim - 1)
        slowed = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        frequencies = frequencies * (1 - slowed * (1 - 1 / stretch))
        factor = 0.1 * math.log(stretch) + 1.0
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"rotary_frequencies: scaling {scaling!r} is none of 'none', 'linear', 'ntk', 'yarn'")
    return frequencies.to(device) if device is not None else frequencies, factor


_NONE = (0, 0)


def _half(name: str, x: torch.Tensor, out: Optional[torch.Tensor], like: tuple) -> tuple:
    """Checks queries or keys and their output: (heads, output, strides of x, strides of the output, addresses of both)."""
    dtype, tokens, dim, device, size = like
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim:
        raise ValueError(f"rotate_rows: {name} must be [{tokens}, heads, {dim}], got {tuple(shape)}")
    if x.dtype != dtype or x.device != device:
        raise ValueError(f"rotate_rows: {name} must be {dtype} on {device}")
    if stride[2] != 1 and dim > 1:
        raise _native.NotCovered(f"rotate_rows: {name} must have a unit stride over the head dim")
    heads, at, to = shape[1], x.data_ptr(), stride
    out_at = at
    if out is None:
        out = x
    elif out is not x:
        if out.shape != shape or out.dtype != dtype or out.device != device:
            raise ValueError(f"rotate_rows: {name}_out must have {name}'s shape, dtype and device")
        to, out_at = out.stride(), out.data_ptr()
        if to[2] != 1 and dim > 1:
            raise _native.NotCovered(f"rotate_rows: {name}_out must have a unit stride over the head dim")
        if tokens and heads and (at != out_at or to != stride):
            span = ((tokens - 1) * stride[0] + (heads - 1) * stride[1] + dim) * size
            if at < out_at + ((tokens - 1) * to[0] + (heads - 1) * to[1] + dim) * size and out_at < at + span:
                layout = lambda strides: ((tokens, strides[0] * size), (heads, strides[1] * size))  # noqa: E731
                if not _native.apart(at, layout(stride), dim * size, out_at, layout(to), dim * size):
                    raise ValueError(f"rotate_rows: {name}_out may be {name} itself, but not overlap it otherwise")
    (near, count), (far, others) = ((to[1], heads), (to[0], tokens)) if to[1] <= to[0] else ((to[0], tokens), (to[1], heads))
    if tokens and heads and ((count > 1 and near < dim) or (others > 1 and far < (near * (count - 1) if count > 1 else 0) + dim)):
        raise ValueError(f"rotate_rows: heads of the output of {name} overlap: every one needs its own storage")
    return heads, out, stride, to, at, out_at


def rotate_rows(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    interleaved: bool = False,
    factor: float = 1.0,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns the first ``2 len(frequencies)`` elements of every head by its row's position, in place without outputs.

    ``q`` [tokens, heads, D] and ``k`` [tokens, kv_heads, D] (None: queries alone) in bf16, fp16 or fp32, any strides
    over tokens and heads (so the parts of one packed projection); ``positions`` [tokens] int32 / int64; ``frequencies`` fp64
    radians a position, at most 512. Pair ``i`` is the elements ``(i, half + i)``, or ``(2 i, 2 i + 1)`` where ``interleaved``:
    ``(x, y) -> factor (x cos - y sin, y cos + x sin)`` of ``position * frequencies[i]``. The elements behind the turned ones
    are copied. Outputs for both or for neither; what is written is memory that no other argument has. Angles are computed in 64
    bits, products in 32, each element rounded once to the rows' dtype. Returns ``(q_out, k_out)``.
    """
    code = _DTYPES.get(q.dtype)
    if code is None:
        raise _native.NotCovered(f"rotate_rows: rows must be bf16, fp16 or fp32, got {q.dtype}")
    if q.dim() != 3:
        raise ValueError(f"rotate_rows: q must be [tokens, heads, D], got {tuple(q.shape)}")
    (tokens, _, dim), device = q.shape, q.device
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous() or frequencies.device != device:
        raise ValueError(f"rotate_rows: frequencies must be a contiguous fp64 vector on {device}")
    half = frequencies.shape[0]
    if not 0 < half <= 512 or 2 * half > dim:
        raise ValueError(f"rotate_rows: {half} pairs do not fit heads of {dim} (at most 512 pairs)")
    if positions.dim() != 1 or positions.shape[0] < tokens or positions.device != device:
        raise ValueError(f"rotate_rows: positions must be [{tokens}] on {device}")
    if k is None and k_out is not None:
        raise ValueError("rotate_rows: k_out without k")
    like = (q.dtype, tokens, dim, device, 4 if code == _native.F32 else 2)
    heads, q_out, qs, qo, q_at, qo_at = _half("q", q, q_out, like)
    kv_heads, ks, ko, k_at, ko_at = 0, _NONE, _NONE, None, None
    if k is not None:
        kv_heads, k_out, ks, ko, k_at, ko_at = _half("k", k, k_out, like)
        if (q_at == qo_at) != (k_at == ko_at) and heads and kv_heads:
            raise ValueError("rotate_rows: q_out and k_out go together")
    if tokens == 0:
        return q_out, k_out
    args = _native.RotaryArgs(q_at, k_at, qo_at, ko_at, qs[0], qs[1], ks[0], ks[1], qo[0], qo[1], ko[0], ko[1],
                              _native.itab(positions), frequencies.data_ptr(), factor, tokens, heads, kv_heads, dim, half, interleaved,
                              code)
    _native.launch("eagle4_rotary", args, device)
    return q_out, k_out
