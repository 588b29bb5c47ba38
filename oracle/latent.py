"""Attention over latent rows in 64 bits, request by request, with the bound that 16-bit weights allow."""

from __future__ import annotations

import torch


def latent_attention(q, new, cache, table, context, starts, masks, scale, rank, page_scale=None):
    """``(out, bound)`` [tokens, heads, rank] fp64. ``bound`` holds for a kernel that rounds each weight and each output to
    ``q``'s dtype (relative error u, half its eps) and sums scores in fp32: with A = sum_k w_k |c_k|,
    ``u (|o| + A) + 2 d A``, where d bounds a score's absolute error (dim additions, each at most 2^-24 of the sum of the
    terms' sizes, and the product with the scale), and fp16's smallest weights, 2^-25 each at worst, times the largest |c|."""
    tokens, heads, dim = q.shape
    out = torch.zeros(tokens, heads, rank, dtype=torch.float64)
    bound = torch.zeros_like(out)
    u = torch.finfo(q.dtype).eps / 2
    blocks, page, _ = cache.shape
    for b in range(len(starts) - 1):
        lo, width = int(starts[b]), int(starts[b + 1]) - int(starts[b])
        held = []
        for k in range(int(context[b])):
            block = int(table[b, k // page])
            if 0 <= block < blocks:
                row = cache[block, k % page].double()
                held.append(row if page_scale is None else row * float(page_scale[block]))
        for r in range(width):
            keys = held + [new[lo + j].double() for j in range(width) if int(masks[b, r]) >> j & 1]
            if not keys:
                continue
            c = torch.stack(keys)
            qr = q[lo + r].double()
            w = torch.softmax(qr @ c.t() * scale, -1)
            out[lo + r] = w @ c[:, :rank]
            size = w @ c[:, :rank].abs()
            d = (dim + 4) * 2.0 ** -24 * float((qr.abs() @ c.abs().t()).max()) * abs(scale)
            tiny = 0.0 if q.dtype == torch.bfloat16 else len(keys) * 2.0 ** -25 * float(c[:, :rank].abs().max())
            bound[lo + r] = u * (out[lo + r].abs() + size) + 2 * d * size + tiny + 1e-30
    return out, bound
