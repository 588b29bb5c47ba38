"""Tree acceptance by sampling, in 64 bits, row by row: what ``sample_tree`` leaves for given uniform numbers."""

from __future__ import annotations

import numpy as np


def distribution(logits: np.ndarray, temperature: float) -> tuple[np.ndarray, bool]:
    """``softmax(logits / temperature)`` in 64 bits, and whether all mass is on the argmax (temperature not above 0, or a
    maximum that is not finite; NaN is the largest value, the first index wins)."""
    x = logits.astype(np.float64)
    top = np.max(x)  # NaN if any is
    if not temperature > 0 or not np.isfinite(top):
        p = np.zeros_like(x)
        p[int(np.argmax(np.isnan(x))) if np.isnan(x).any() else int(np.argmax(x))] = 1.0
        return p, True
    with np.errstate(invalid="ignore"):
        e = np.exp(np.where(np.isneginf(x), -np.inf if np.isfinite(temperature) else 0.0, (x - top) / temperature))
    if not np.isfinite(temperature):
        e = np.where(np.isneginf(x), 0.0, 1.0)
    return e / e.sum(), False


def walk(logits, drafted, parents, coins, final_coin, temperature, probs=None):
    """One request: ``logits [rows, vocab]``, ``drafted [rows]``, ``parents [rows]``, ``coins [rows]`` -> (tokens, path)."""
    rows, vocab = logits.shape
    node, tokens, path = 0, [], [0]
    if rows == 0:
        return [], []
    while True:
        p, single = distribution(logits[node], temperature)
        left, mass, spent, following = p.copy(), 1.0, 0.0, -1
        for child in range(1, rows):
            if parents[child] != node or len(path) >= rows:
                continue
            x = int(drafted[child])
            if not 0 <= x < vocab:
                continue
            if single:
                if p[x] == 1.0:
                    following = child
                    break
                continue
            q = 1.0 if probs is None else float(probs[node, x])
            if float(coins[child]) * q * mass < left[x]:
                following = child
                break
            if probs is None:
                left[x] = 0.0
            else:
                spent += mass
                r = p - spent * probs[node].astype(np.float64)
                left = np.where(np.isnan(r), 0.0, np.maximum(r, 0.0))
            mass = left.sum()
        if following >= 0:
            tokens.append(int(drafted[following]))
            path.append(following)
            node = following
            continue
        if not mass > 0:
            left = p
        running = np.cumsum(left)
        at = int(np.searchsorted(running, float(final_coin) * running[-1], side="right")) if final_coin == final_coin else vocab
        tokens.append(at if at < vocab else int(np.flatnonzero(left > 0)[-1]))
        return tokens, path


def sample_tree(logits, drafted, cu_num_logits, idx_mapping, parents, coins, final_coins, temperature, path, path_len, width,
                probs=None):
    """The batch's walks: ``(sampled [R, width] filled with -1, num_sampled [R])``; ``path`` / ``path_len`` in place."""
    logits = logits.float().numpy()
    probs = None if probs is None else probs.float().numpy()
    cu = [int(x) for x in cu_num_logits]
    sampled = np.full((len(cu) - 1, width), -1, dtype=np.int64)
    count = np.zeros(len(cu) - 1, dtype=np.int32)
    for b in range(len(cu) - 1):
        rows = min(cu[b + 1] - cu[b], width)
        sl, slot = slice(cu[b], cu[b] + rows), int(idx_mapping[b])
        tokens, taken = walk(logits[sl], drafted[sl].numpy(), parents[slot].numpy(), coins[sl].numpy(), float(final_coins[b]),
                             float(temperature[b]), None if probs is None else probs[sl])
        sampled[b, : len(tokens)] = tokens
        count[b] = len(tokens)
        path[slot, : len(taken)] = path.new_tensor(taken)
        path_len[slot] = len(taken)
    return sampled, count
