"""Performance cases of a sampled draft step over quantized pages, each operator in its plain torch form and as the package's
calls (``own``).

A case is a dict of plain values with a ``kind``:

- ``draw``: tokens drawn from a draft's rows under temperature, top-k, top-p and min-p, with or without the distribution
  that they were drawn from (``draw_tokens``);
- ``truncate``: a target's rows with the tokens that those rules leave out at -inf, for the sampled walk (``truncate_logits``);
- ``rotary``: queries and keys rotated by their positions (``rotate_rows``);
- ``tables``: block tables grown for a round's or a prompt's rows, their slots, and the pages given back (``resize_tables``,
  ``slot_maps``);
- ``rows``: a draft step's or a draft extend's attention over fp8 pages with a scale per (page, head) (``rows_attention``).
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import torch

own = False

PACKAGE = str(Path(__file__).resolve().parent.parent / "eagle-4_amd")
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"": 0, "bf16": 2, "f16": 2, "f32": 4}
E4M3_MAX = 448.0


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user's draft step: the next token of one row
        dict(name="draw_b1", kind="draw", batch=1, rows=1, draws=1, vocab=151936, dtype="bf16", probs="", flat=False),
        # the serving batch's draft step: four frontier rows a request, two children each, drawn with their probabilities
        dict(name="draw_probs_b64", kind="draw", batch=64, rows=4, draws=2, vocab=151936, dtype="bf16", probs="f32", flat=False),
        # the first tokens of joining requests, fp32 logits over an odd vocabulary, high temperatures without a top-k
        dict(name="draw_flat_f32", kind="draw", batch=24, rows=1, draws=1, vocab=50257, dtype="f32", probs="", flat=True),
        # the target's rows of one user's tree
        dict(name="truncate_b1", kind="truncate", batch=1, rows=16, vocab=151936, dtype="bf16", flat=False),
        # the target's rows of the serving batch's trees
        dict(name="truncate_b64", kind="truncate", batch=64, rows=16, vocab=151936, dtype="bf16", flat=False),
        # one user's tree: part of each head rotated, halves paired
        dict(name="rotary_b1", kind="rotary", tokens=16, hq=24, hkv=4, d=256, part=64, paired=False, dtype="bf16", base=1e7,
             stretch=1.0, far=8192),
        # a chunk of long prompts, whole heads, neighbours paired, positions stretched for a long context
        dict(name="rotary_prompt", kind="rotary", tokens=8191, hq=32, hkv=8, d=128, part=128, paired=True, dtype="bf16",
             base=1e4, stretch=8.0, far=262144),
        # a round's rows of the serving batch
        dict(name="tables_round_b64", kind="tables", batch=64, page=16, nmin=8, nmax=16, lmin=512, lmax=8192),
        # prompts that join, in an odd page size
        dict(name="tables_prompt_b96", kind="tables", batch=96, page=24, nmin=1, nmax=4096, lmin=0, lmax=512),
        # one user's draft step over the whole context
        dict(name="rows_fp8_b1", kind="rows", batch=1, rows=4, step=3, window=0, length=4096, hq=32, hkv=8, d=128, page=16,
             dtype="bf16"),
        # the serving batch's draft step over a sliding window
        dict(name="rows_fp8_step_b64", kind="rows", batch=64, rows=4, step=7, window=4096, length=8192, hq=32, hkv=8, d=128,
             page=16, dtype="bf16"),
        # a draft extend after a round, wide heads
        dict(name="rows_fp8_extend_b32", kind="rows", batch=32, rows=9, step=0, window=2048, length=6000, hq=24, hkv=4, d=256,
             page=16, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between ``lo`` and ``hi``, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(("draw", "draw", "truncate", "truncate", "rotary", "tables", "rows", "rows", "rows"))
        if kind in ("draw", "truncate"):
            case = dict(kind=kind, batch=_log(rng, 1, 256), rows=rng.randint(1, 8 if kind == "draw" else 32),
                        vocab=rng.choice((151936, 151936, 50257, 32000, rng.randint(300, 5000))),
                        dtype=rng.choice(("bf16", "bf16", "f16", "f32")), flat=rng.random() < 0.3)
            if kind == "draw":
                case.update(draws=rng.choice((1, 1, 2, 5)), probs=rng.choice(("", "", "f32", "bf16")))
        elif kind == "rotary":
            d, part = rng.choice(((256, 64), (128, 128), (64, 64), (128, 32), (576, 64)))
            hq, hkv = rng.choice(((24, 4), (32, 8), (16, 1), (8, 2), (128, 1)))
            case = dict(kind=kind, tokens=_log(rng, 1, 8192), hq=hq, hkv=hkv, d=d, part=part, paired=rng.random() < 0.5,
                        dtype=rng.choice(("bf16", "bf16", "f16", "f32")), base=rng.choice((1e4, 5e5, 1e7)),
                        stretch=rng.choice((1.0, 4.0, 40.0)), far=_log(rng, 4, 1 << 20))
        elif kind == "tables":
            nmax = _log(rng, 1, 4096)
            lmax = _log(rng, 1, 16384)
            case = dict(kind=kind, batch=_log(rng, 1, 512), page=rng.choice((16, 16, 64, 24, 1)), nmin=max(0, nmax // 3), nmax=nmax,
                        lmin=lmax // rng.choice((1, 4, 50)), lmax=lmax)
        else:
            hq, hkv, d = rng.choice(((32, 8, 128), (16, 4, 128), (8, 2, 64), (24, 4, 256), (16, 16, 64)))
            step = rng.choice((0, rng.randint(1, 11)))
            case = dict(kind=kind, batch=_log(rng, 1, 96), rows=rng.randint(1, 16 if step == 0 else 8), step=step,
                        window=rng.choice((0, 0, 2048, 1000)), length=_log(rng, 3, 16384), hq=hq, hkv=hkv, d=d,
                        page=rng.choice((16, 16, 64, 24)), dtype=rng.choice(("bf16", "bf16", "f16")))
        if _affordable(case):
            return case


def _affordable(c):
    """No more work, and no larger padded arrays, than the largest listed case of its kind."""
    if c["kind"] in ("draw", "truncate"):
        return c["batch"] * c["rows"] * c["vocab"] * (4 if c.get("probs") else 1) <= 1024 * 151936
    if c["kind"] == "rotary":
        return c["tokens"] * (c["hq"] + c["hkv"]) * c["d"] * BYTES[c["dtype"]] <= 8192 * 40 * 128 * 2
    if c["kind"] == "tables":
        return c["batch"] * c["nmax"] <= 96 * 4096 and c["batch"] * (c["lmax"] + c["nmax"]) // c["page"] <= 1 << 18
    w = min(c["length"], c["window"] or c["length"]) + c["rows"]
    return (c["batch"] * w * c["hkv"] * c["d"] <= 64 * 4200 * 1024
            and c["batch"] * w * c["hq"] * c["rows"] <= 64 * 4200 * 32 * 4)


# ---- sizes -------------------------------------------------------------------------------------------------------------
def _sizes(c):
    """Rows and context of every request, as lists over the batch: the case alone gives them, so that every seed's outputs
    have one shape."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    if c["kind"] == "tables":
        context = [rng.randint(c["lmin"], c["lmax"]) for _ in range(c["batch"])]
        return [rng.randint(c["nmin"], c["nmax"]) for _ in context], context
    if c["kind"] == "truncate":  # trees of different sizes
        return [rng.randint(max(1, c["rows"] // 2), c["rows"]) if c["batch"] > 1 else c["rows"] for _ in range(c["batch"])], None
    if c["kind"] == "draw":
        return [c["rows"]] * c["batch"], None
    return [c["rows"]] * c["batch"], [rng.randint(max(1, c["length"] // 2), c["length"]) for _ in range(c["batch"])]


def work(case):
    """What a pass cannot do without: every input read once, every output written once."""
    c = case
    if c["kind"] in ("draw", "truncate"):
        values = sum(_sizes(c)[0]) * c["vocab"]
        out = BYTES[c["probs"]] if c["kind"] == "draw" else BYTES[c["dtype"]]
        return {"bytes": values * (BYTES[c["dtype"]] + out), "flops": values * 4.0}
    if c["kind"] == "rotary":
        values = c["tokens"] * (c["hq"] + c["hkv"])
        return {"bytes": values * c["d"] * 2 * BYTES[c["dtype"]] + 8 * c["tokens"], "flops": values * c["part"] * 3.0}
    counts, context = _sizes(c)
    if c["kind"] == "tables":
        held = sum(-(-(n + k) // c["page"]) for n, k in zip(counts, context))
        new = held - sum(-(-k // c["page"]) for k in context)
        return {"bytes": 8 * sum(counts) + 4 * 2 * held + 4 * 4 * new + 24 * c["batch"], "flops": float(sum(counts) + held)}
    keys = sum(min(k, c["window"] or k) for k in context)
    keys += c["batch"] * (c["rows"] if c["step"] == 0 else c["rows"] * c["step"])
    rows = c["batch"] * c["rows"]
    return {"bytes": keys * c["hkv"] * c["d"] * 2 + 4 * keys // c["page"] + rows * c["hq"] * c["d"] * 4,
            "flops": 4.0 * c["rows"] * c["hq"] * c["d"] * keys}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _pages(rng, lens, page):
    """A block table for ``lens`` positions a request, over pages in an order of their own, and the number of pages."""
    need = [max(1, -(-int(n) // page)) for n in lens]
    total = sum(need) + 3
    order = np.random.RandomState(rng.randrange(1 << 30)).permutation(total)
    table = np.zeros((len(lens), max(need) + 1), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    return table, total


def _cache(gen, dev, blocks, page, heads, dim):
    """fp8 pages of values whose size differs from page to page, and the scales that amax / 448 gives."""
    size = 0.25 + 1.5 * torch.rand(blocks, 1, heads, 1, generator=gen, device=dev)
    x = torch.randn(blocks, page, heads, dim, generator=gen, device=dev) * size
    scale = x.abs().amax((1, 3)) / E4M3_MAX
    return (x / scale[:, None, :, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    rng = random.Random(int(seed) * 7919 + 29)
    gen = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    make = {"draw": _prepare_draw, "truncate": _prepare_draw, "rotary": _prepare_rotary, "tables": _prepare_tables,
            "rows": _prepare_rows}[c["kind"]]
    return make(c, rng, gen, dev, on)


def _prepare_draw(c, rng, gen, dev, on):
    counts, vocab = np.array(_sizes(c)[0]), c["vocab"]
    rows = int(counts.sum())
    # a language model's logits: a broad floor and some two dozen likely tokens
    floor = 4.2 * math.sqrt(math.log(vocab) / math.log(151936))
    logits = torch.randn(rows, vocab, generator=gen, device=dev) * (0.45 * floor)
    step = vocab // 24  # one of each stretch, so that no token comes twice
    likely = step * torch.arange(24, device=dev) + torch.randint(0, step, (rows, 24), generator=gen, device=dev)
    logits.scatter_(1, likely, math.log(vocab) + 0.6 + 1.5 * torch.randn(rows, 24, generator=gen, device=dev))
    # the requests' own settings, as users mix them: a few are greedy, some rules are off
    pick = lambda values: on(np.array([rng.choice(values) for _ in range(c["batch"])]))  # noqa: E731
    hot = (0.9, 1.0, 1.3) if c["flat"] else (0.6, 0.7, 0.8, 1.0)
    temperature = pick(hot * 4 + (0.0,)).float()
    top_k = pick((0, 0, 0, 50) if c["flat"] else (20, 20, 50, 200, 0)).int()
    top_p = pick((0.8, 0.9, 0.95, 1.0)).float()
    min_p = pick((0.0, 0.0, 0.0, 0.02, 0.1)).float()
    entries = on(np.repeat(np.arange(c["batch"], dtype=np.int32), counts))
    coins = probs = None
    if c["kind"] == "draw":
        coins = torch.rand(rows, c["draws"], generator=gen, device=dev)
        probs = torch.empty(rows, vocab, dtype=DTYPES[c["probs"]], device=dev) if c["probs"] else None
    return SimpleNamespace(kind=c["kind"], logits=logits.to(DTYPES[c["dtype"]]), coins=coins, temperature=temperature,
                           top_k=top_k, top_p=top_p, min_p=min_p, entries=entries, probs=probs)


def _frequencies(c):
    """Radians per position of every pair, in 64 bits."""
    half = c["part"] // 2
    return c["base"] ** (-np.arange(half) / half) / c["stretch"]


def _prepare_rotary(c, rng, gen, dev, on):
    dt = DTYPES[c["dtype"]]
    rows = lambda heads: torch.randn(c["tokens"], heads, c["d"], generator=gen, device=dev).to(dt)  # noqa: E731
    q, k = rows(c["hq"]), rows(c["hkv"])
    start = rng.randrange(max(1, c["far"] - c["tokens"]))
    positions = start + torch.arange(c["tokens"], device=dev)
    return SimpleNamespace(kind="rotary", q=q, k=k, positions=positions, frequencies=on(_frequencies(c)), paired=c["paired"],
                           factor=1.0 + 0.1 * math.log(c["stretch"]), q_out=torch.empty_like(q), k_out=torch.empty_like(k))


def _prepare_tables(c, rng, gen, dev, on):
    counts, context = (np.array(x, dtype=np.int32) for x in _sizes(c))
    b, page = c["batch"], c["page"]
    held, need = -(-context // page), -(-(context + counts) // page)
    width = int(need.max()) + 1
    total = int(need.sum()) + 5
    order = np.random.RandomState(rng.randrange(1 << 30)).permutation(total).astype(np.int32)
    slots = np.array(rng.sample(range(b + 3), b), dtype=np.int32)
    table, pages = np.zeros((b + 3, width), dtype=np.int32), np.zeros(b + 3, dtype=np.int32)
    at = 0
    for i, n in enumerate(held):
        table[slots[i], :n] = order[at : at + n]
        pages[slots[i]] = n
        at += n
    free = np.zeros(total, dtype=np.int32)
    free[: total - at] = order[at:]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return SimpleNamespace(kind="tables", table=on(table), pages=on(pages), idx=on(slots), context=on(context), page=page,
                           lens=on(context + counts), starts=on(starts), free=on(free), num_free=on(np.array([total - at], np.int32)),
                           slots=torch.empty(max(1, int(starts[-1])), dtype=torch.int64, device=dev),
                           batch_table=torch.empty(b, width, dtype=torch.int32, device=dev))


def _prepare_rows(c, rng, gen, dev, on):
    b, r, step, page, dt = c["batch"], c["rows"], c["step"], c["page"], DTYPES[c["dtype"]]
    context = np.array(_sizes(c)[1], dtype=np.int32)
    added = r * step if step else r  # nodes drafted so far, or the extend's rows, behind the context
    table, blocks = _pages(rng, context + added, page)
    keys, k_scale = _cache(gen, dev, blocks, page, c["hkv"], c["d"])
    values, v_scale = _cache(gen, dev, blocks, page, c["hkv"], c["d"])
    ancestors = None
    if step:
        levels = np.random.RandomState(rng.randrange(1 << 30)).randint(0, r, (b, r, step)) + r * np.arange(step)
        at = context[:, None, None] + levels
        ancestors = on((table[np.arange(b)[:, None, None], at // page] * page + at % page).astype(np.int32))
    units = 4 * torch.cuda.get_device_properties(dev).multi_processor_count
    splits = max(8, 2 ** max(0, round(math.log2(units / (b * c["hq"])))))
    padded = max(16, 1 << (r - 1).bit_length())
    parts = b * c["hq"] * (splits + 1) * padded
    q = torch.randn(b * r, c["hq"], c["d"], generator=gen, device=dev).to(dt)
    return SimpleNamespace(kind="rows", q=q, keys=keys, values=values, k_scale=k_scale, v_scale=v_scale, table=on(table),
                           seq=on(context), longest=int(context.max()), ancestors=ancestors, rows=r, step=step,
                           window=c["window"], page=page, scale=c["d"] ** -0.5, splits=splits, out=torch.empty_like(q),
                           part_out=torch.empty(parts, c["d"], device=dev), part_lse=torch.empty(parts, device=dev))


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        return _call(s)
    return {"draw": _draw, "truncate": _truncate, "rotary": _rotary, "tables": _tables, "rows": _rows}[s.kind](s)


def _call(s):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    if s.kind == "draw":
        from eagle_harness.vllm.sampling import draw_tokens

        tokens = draw_tokens(s.logits, s.coins, s.temperature, s.top_k, s.top_p, s.min_p, entries=s.entries, probs=s.probs)
        return tokens, s.probs
    if s.kind == "truncate":
        from eagle_harness.vllm.sampling import truncate_logits

        return truncate_logits(s.logits, s.temperature, s.top_k, s.top_p, s.min_p, entries=s.entries)
    if s.kind == "rotary":
        from eagle_harness.vllm.rotary import rotate_rows

        return rotate_rows(s.q, s.k, s.positions, s.frequencies, interleaved=s.paired, factor=s.factor, q_out=s.q_out,
                           k_out=s.k_out)
    if s.kind == "tables":
        from eagle_harness.vllm.page_tables import resize_tables, slot_maps

        resize_tables(s.table, s.pages, s.idx, s.lens, s.free, s.num_free, s.page)
        slots, batch_table = slot_maps(s.table, s.pages, s.idx, s.context, s.starts, s.page, slots=s.slots,
                                       batch_table=s.batch_table)
        resize_tables(s.table, s.pages, s.idx, s.context, s.free, s.num_free, s.page)  # what no accepted row needs
        return slots, batch_table, s.pages, s.free, s.num_free
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention

    rows_attention(s.q, s.keys, s.values, s.out, s.part_out, s.part_lse, s.table, s.seq, s.ancestors, rows_per_request=s.rows,
                   step=s.step, window=s.window, scale=s.scale, launch=RowsLaunch(splits=s.splits, block_n=32),
                   table_page=s.page, k_scale=s.k_scale, v_scale=s.v_scale)
    return s.out


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _kept(s):
    """The rows' tokens in their order (logits descending, the lower index first among equals), their masses and running
    masses in 64 bits, and how many each row keeps."""
    of = s.entries.long()
    t, k, p, m = (v[of][:, None] for v in (s.temperature.double(), s.top_k.long(), s.top_p.double(), s.min_p.double()))
    x, order = torch.sort(s.logits.float(), dim=1, descending=True, stable=True)
    at = torch.arange(x.shape[1], device=x.device)[None]
    greedy = t <= 0
    x = x.double()
    mass = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, t))
    mass = torch.where(greedy, (at == 0).double(), mass)
    most = torch.where(k > 0, k, x.shape[1]).clamp(max=x.shape[1])
    most = torch.minimum(most, (mass >= m).sum(1, keepdim=True)).clamp(min=1)
    run = torch.cumsum(mass, 1)
    limit = p * run.gather(1, most - 1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], 1)
    count = ((at < most) & ((before < limit) | (p >= 1))).sum(1, keepdim=True).clamp(min=1)
    return order, mass, run, count, torch.where(greedy, 1, count)


def _draw(s):
    order, mass, run, _, count = _kept(s)
    total = run.gather(1, count - 1)
    at = torch.searchsorted(run, s.coins.double() * total, right=True)
    tokens = order.gather(1, torch.minimum(at, count - 1))
    if s.probs is None:
        return tokens, None
    kept = torch.arange(run.shape[1], device=run.device)[None] < count
    share = torch.where(kept, mass / total, 0.0)
    return tokens, torch.zeros_like(mass).scatter_(1, order, share).to(s.probs.dtype)


def _truncate(s):
    order, _, _, _, count = _kept(s)
    kept = torch.arange(order.shape[1], device=order.device)[None] < count
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    return torch.where(kept, s.logits, -math.inf)


def _rotary(s):
    angle = s.positions.double()[:, None] * s.frequencies[None]
    c, d = (torch.cos(angle) * s.factor).float()[:, None], (torch.sin(angle) * s.factor).float()[:, None]
    half = s.frequencies.shape[0]

    def turned(x):
        x = x.float()
        part, rest = x[..., : 2 * half], x[..., 2 * half :]
        a, b = (part[..., 0::2], part[..., 1::2]) if s.paired else (part[..., :half], part[..., half:])
        a, b = a * c - b * d, b * c + a * d
        return torch.cat([torch.stack([a, b], -1).flatten(-2) if s.paired else torch.cat([a, b], -1), rest], -1)

    return turned(s.q).to(s.q.dtype), turned(s.k).to(s.k.dtype)


def _resized(table, pages, idx, lens, free, num_free, page):
    """Tables, page counts and free pages after giving back (the last request's last page first) and taking."""
    idx, dev = idx.long(), table.device
    have, need = pages[idx].long(), (lens.long() + page - 1) // page
    back, more = (have - need).clamp(min=0), (need - have).clamp(min=0)
    first = torch.cumsum(back, 0) - back  # of the returned pages, counted from the top
    entry = torch.arange(table.shape[1], device=dev)[None]
    given = (entry >= need[:, None]) & (entry < have[:, None])
    top = num_free.long() + back.sum()
    held = table[idx].long()
    spot = torch.where(given, top - 1 - (first[:, None] + entry - need[:, None]), free.shape[0])
    stack = torch.cat([free, free[:1]]).long().scatter(0, spot.flatten(), held.flatten())
    ends = torch.cumsum(more, 0)
    served = (more > 0) & (ends <= top)
    taken = served[:, None] & (entry >= have[:, None]) & (entry < need[:, None])
    source = (top - 1 - ((ends - more)[:, None] + entry - have[:, None])).clamp(min=0, max=free.shape[0])
    held = torch.where(taken, stack[source], held)
    pages = pages.scatter(0, idx, torch.where(served | (back > 0), need, have).to(pages.dtype))
    left = top - torch.where(served, more, 0).sum()
    return table.index_copy(0, idx, held.to(table.dtype)), pages, stack[:-1].to(free.dtype), left.to(num_free.dtype)


def _tables(s):
    table, pages, free, num_free = _resized(s.table, s.pages, s.idx, s.lens, s.free, s.num_free, s.page)
    idx, dev = s.idx.long(), table.device
    row = torch.arange(s.slots.shape[0], device=dev)
    request = (torch.searchsorted(s.starts.long(), row, right=True) - 1).clamp(max=idx.shape[0] - 1)
    position = s.context.long()[request] + row - s.starts.long()[request]
    entry = position // s.page
    good = (entry < pages[idx].long()[request]) & (row < s.starts[-1])
    block = table[idx[request], entry.clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(good, block * s.page + position % s.page, -1)
    held = torch.arange(table.shape[1], device=dev)[None] < pages[idx][:, None]
    batch_table = torch.where(held, table[idx], 0)
    _, pages, free, num_free = _resized(table, pages, s.idx, s.context, free, num_free, s.page)
    return slots, batch_table, pages, free, num_free


def _rows(s):
    b, r = s.seq.shape[0], s.rows
    dev, (hkv, d) = s.q.device, s.keys.shape[2:]
    group = s.q.shape[1] // hkv
    seq = s.seq.long()
    last = seq - 1 if s.step else seq + r - 1
    first = (seq - 1 if s.step else seq) - (s.window - 1)
    first = first.clamp(min=0) if s.window > 0 else torch.zeros_like(seq)
    span = s.longest + (0 if s.step else r)
    if s.window > 0:
        span = min(span, s.window + (0 if s.step else r - 1))
    at = first[:, None] + torch.arange(span, device=dev)[None]  # [b, span]
    inside = at <= last[:, None]
    at = torch.minimum(at, last[:, None])
    block = s.table[torch.arange(b, device=dev)[:, None], at // s.page].long()
    get = lambda x, scale, blk, pos: x.float()[blk, pos] * scale[blk][..., None]  # noqa: E731
    keys, values = get(s.keys, s.k_scale, block, at % s.page), get(s.values, s.v_scale, block, at % s.page)
    q = s.q.float().view(b, r, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, r * group, d).contiguous()
    score = torch.matmul(q, keys.permute(0, 2, 3, 1).contiguous()).view(b, hkv, r, group, span) * s.scale
    row = torch.arange(r, device=dev)
    seen = inside[:, None].expand(-1, r, -1)
    if not s.step:
        pos = seq[:, None] + row[None]
        seen = seen & (at[:, None] <= pos[..., None])
        if s.window > 0:
            seen = seen & (at[:, None] > pos[..., None] - s.window)
    score = torch.where(seen[:, None, :, None], score, -math.inf)
    if s.step:
        blk, pos = s.ancestors.long() // s.page, s.ancestors.long() % s.page  # [b, r, step]
        own_keys, own_values = get(s.keys, s.k_scale, blk, pos), get(s.values, s.v_scale, blk, pos)  # [b, r, step, hkv, d]
        own_score = (q.view(b, hkv, r, group, 1, d) * own_keys.permute(0, 3, 1, 2, 4)[:, :, :, None]).sum(-1) * s.scale
        score = torch.cat([score, own_score], -1)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    total = weight.sum(-1, keepdim=True)
    got = torch.matmul(weight[..., :span].reshape(b, hkv, r * group, span), values.permute(0, 2, 1, 3).contiguous())
    got = got.view(b, hkv, r, group, d)
    if s.step:
        got = got + (weight[..., span:, None] * own_values.permute(0, 3, 1, 2, 4)[:, :, :, None]).sum(-2)
    got = (got / total).permute(0, 2, 1, 3, 4).reshape(b * r, hkv * group, d)
    return s.out.copy_(got)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s.kind in ("draw", "truncate"):
        if s.kind == "draw" and s.probs is None:
            return None
        got = torch.stack([_exact_row(s, n) for n in range(s.logits.shape[0])])
        return (None, got) if s.kind == "draw" else got
    if s.kind == "rotary":
        return _exact_rotary(s, s.q), _exact_rotary(s, s.k)
    if s.kind == "tables":
        return None
    return _exact_rows(s)


def _exact_row(s, n):
    """One row's distribution, or its logits with -inf for what is left out."""
    x, i = s.logits[n].double(), int(s.entries[n])
    t, k, p, m = (float(v[i]) for v in (s.temperature, s.top_k, s.top_p, s.min_p))
    if t <= 0:
        keep = torch.zeros_like(x, dtype=torch.bool)
        keep[int(torch.nonzero(x == x.max())[0])] = True
    else:
        logp = torch.log_softmax(x / t, 0)
        order = torch.argsort(-x, stable=True)
        if m > 0:
            order = order[torch.exp(logp[order] - logp.max()) >= m]
        if k > 0:
            order = order[: int(k)]
        share = torch.softmax(x[order] / t, 0)
        ahead = torch.cumsum(share, 0) - share
        if p < 1:
            order = order[(ahead < p) | (torch.arange(len(order), device=x.device) == 0)]
        keep = torch.zeros_like(x, dtype=torch.bool)
        keep[order] = True
    if s.kind == "truncate":
        return torch.where(keep, x, -math.inf)
    got = torch.zeros_like(x)
    got[keep] = torch.softmax(x[keep] / t, 0) if t > 0 else 1.0
    return got


def _exact_rotary(s, x):
    half = s.frequencies.shape[0]
    turn = s.factor * torch.exp(1j * (s.positions.double()[:, None] * s.frequencies[None]))[:, None]
    x = x.double().clone()
    even, odd = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s.paired else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., even], x[..., odd]) * turn
    x[..., even], x[..., odd] = z.real, z.imag
    return x


def _exact_rows(s):
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=s.q.device)
    hkv = s.keys.shape[2]
    for b, length in enumerate(s.seq.tolist()):
        for j in range(s.rows):
            last = length - 1 if s.step else length + j
            at = torch.arange(max(0, last - s.window + 1) if s.window > 0 else 0, last + 1, device=out.device)
            slot = s.table[b, at // s.page].long() * s.page + at % s.page
            if s.step:
                slot = torch.cat([slot, s.ancestors[b, j].long()])
            blk, pos = slot // s.page, slot % s.page
            k = s.keys.view(torch.uint8)[blk, pos].view(torch.float8_e4m3fn).double() * s.k_scale[blk].double()[..., None]
            v = s.values.view(torch.uint8)[blk, pos].view(torch.float8_e4m3fn).double() * s.v_scale[blk].double()[..., None]
            q = s.q[b * s.rows + j].double().view(hkv, -1, s.q.shape[2])
            w = torch.softmax((q[:, :, None] * k.permute(1, 0, 2)[:, None]).sum(-1) * s.scale, -1)
            out[b * s.rows + j] = (w[..., None] * v.permute(1, 0, 2)[:, None]).sum(2).reshape(-1, s.q.shape[2])
    return out
