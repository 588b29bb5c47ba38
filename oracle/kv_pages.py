"""fp8-e4m3 pages with one power-of-two scale per (page, head), request by request: writing rows, reading them back."""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def page_scale(amax: float) -> float:
    """The least power of two ``s`` (at least 2^-126) with ``amax <= 448 s``; 0 for 0."""
    if amax == 0:
        return 0.0
    s = 2.0 ** -126
    while amax > E4M3_MAX * s:
        s *= 2.0
    return s


def encode(x: torch.Tensor) -> torch.Tensor:
    """fp64 values to e4m3: the nearest, ties to an even last bit, saturating; NaN stays."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 .. 448, in order
    a = x.abs().clamp(max=E4M3_MAX)
    hi = torch.searchsorted(codes, a.contiguous()).clamp(max=126)  # the first code >= a
    lo = (hi - 1).clamp(min=0)
    up, down = codes[hi] - a, a - codes[lo]
    nearest = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).to(torch.uint8)
    nearest = torch.where(torch.isnan(x), torch.full_like(nearest, 127), nearest)
    sign = torch.signbit(x) & ~torch.isnan(x)
    return (nearest | (sign.to(torch.uint8) << 7)).view(torch.float8_e4m3fn)


def write_rows(rows, cache, scale, table, context: int) -> None:
    """``rows`` [n, heads, D] of one request to positions ``context ..`` of ``table``, in place; ``rows[j]`` None: not
    written. Pages outside the table or the cache are skipped."""
    blocks, page, heads, _ = cache.shape
    done = 0
    while done < len(rows):
        index, lead = (context + done) // page, (context + done) % page
        part = rows[done : done + page - lead]
        done += len(part)
        if index >= len(table) or not 0 <= int(table[index]) < blocks:
            continue
        block = int(table[index])
        for h in range(heads):
            data = [None if r is None else r[h].double() for r in part]
            if all(d is None for d in data):  # no row goes to the page
                continue
            amax = max([float(torch.where(torch.isfinite(d), d.abs(), 0.0).max()) for d in data if d is not None] + [0.0])
            old = float(scale[block, h]) if lead else 0.0
            now = max(old, page_scale(amax))
            if now == 0 and any(bool(torch.isinf(d).any()) for d in data if d is not None):
                now = 1.0  # an infinity saturates at a value, not at 0
            if lead and now > old:
                cache[block, :lead, h] = encode(cache[block, :lead, h].double() * (old / now))
            for j, d in enumerate(data):
                if d is None:
                    continue
                y = d / now if now > 0 else d * 0.0  # (no infinities then)
                cache[block, lead + j, h] = encode(y)
            scale[block, h] = now


def write_pages(key, cache, scale, table, context, starts, path=None, path_len=None, slots=None, max_rows=1 << 30):
    """:func:`write_rows` for every request."""
    for b in range(len(starts) - 1):
        lo, n = int(starts[b]), int(starts[b + 1]) - int(starts[b])
        if path is None:
            rows = [key[lo + j] for j in range(min(n, max_rows))]
        else:
            count = min(int(path_len[int(slots[b])]), path.shape[1], max_rows)
            taken = [int(x) for x in path[int(slots[b]), :count]]
            rows = [key[lo + r] if 0 <= r < n else None for r in taken]
        write_rows(rows, cache, scale, [int(x) for x in table[b]], int(context[b]))


def read_pages(cache, scale, table, starts):
    """Values of every request's first positions, [tokens, heads, D] fp64."""
    blocks, page, heads, dim = cache.shape
    out = torch.zeros(int(starts[-1]), heads, dim, dtype=torch.float64)
    values = cache.double() * scale.double()[:blocks, None, :heads, None]
    for b in range(len(starts) - 1):
        for k in range(int(starts[b + 1]) - int(starts[b])):
            index = k // page
            if index < table.shape[1] and 0 <= int(table[b, index]) < blocks:
                out[int(starts[b]) + k] = values[int(table[b, index]), k % page]
    return out
