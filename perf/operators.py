"""Performance cases of four operators of a sampled or quantized verify round, each in its plain torch form and as the
package's calls (``own``).

A case is a dict of plain values with a ``kind``:

- ``latent``: attention of a round's rows over a paged cache of one latent row a token (``latent_verify_attention``):
  a decode step (width 1), a drafted chain or tree, 16-bit or fp8 pages;
- ``sample``: verification of drafted tokens against the target's probabilities from given uniform numbers
  (``sample_tree``), without and with the draft's own probabilities;
- ``write``: rows quantized into fp8 pages with a scale per (page, head) (``write_kv_pages``): the accepted rows of a
  round, or a prompt's;
- ``read``: rows of fp8 pages gathered back at 16 bits (``read_kv_pages``).

Trees: a node's parent is drawn from the earlier nodes with fewer than 4 children and depth below 12. ``ragged`` gives
the requests trees of different sizes (half the width and up).
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
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
MAX_CHILDREN = 4
E4M3_MAX = 448.0


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    latent = dict(kind="latent", rank=512, rope=64, page=16, dtype="bf16")
    return [
        # one user's decode step over a latent cache with all heads on the card: latency
        dict(latent, name="latent_decode_b1", batch=1, width=1, ragged=False, heads=128, lmin=2048, lmax=2048, cache="bf16"),
        # one user's drafted tree, heads of one rank of eight
        dict(latent, name="latent_tree_b1", batch=1, width=16, ragged=False, heads=16, lmin=4096, lmax=4096, cache="bf16"),
        # the serving batch's trees over prefixes of very different lengths
        dict(latent, name="latent_tree_b64", batch=64, width=16, ragged=True, heads=16, lmin=1024, lmax=8192, cache="bf16"),
        # a large decode batch with short drafted chains over quantized pages
        dict(latent, name="latent_fp8_b128", batch=128, width=4, ragged=False, heads=16, lmin=512, lmax=8192, cache="fp8"),
        # one user's sampled round
        dict(name="sample_b1", kind="sample", batch=1, width=16, chain=False, ragged=False, vocab=151936, dtype="bf16", probs=""),
        # the serving batch's sampled round, trees of the draft's most likely tokens
        dict(name="sample_b64", kind="sample", batch=64, width=16, chain=False, ragged=True, vocab=151936, dtype="bf16", probs=""),
        # chains drawn from a draft model's probabilities
        dict(name="sample_probs_b32", kind="sample", batch=32, width=6, chain=True, ragged=False, vocab=151936, dtype="bf16",
             probs="f32"),
        # fp32 logits over an odd vocabulary, trees whose siblings were drawn independently
        dict(name="sample_probs_tree_f32", kind="sample", batch=12, width=12, chain=False, ragged=True, vocab=50257, dtype="f32",
             probs="f32"),
        # the accepted rows of a serving batch's round, one layer's K and V heads
        dict(name="write_round_b64", kind="write", batch=64, width=16, path=True, heads=4, dim=256, values=True, page=16,
             nmin=16, nmax=16, lmin=512, lmax=4096, dtype="bf16"),
        # a prompt chunk of four requests that join the batch
        dict(name="write_prompt_b4", kind="write", batch=4, width=0, path=False, heads=8, dim=128, values=True, page=16,
             nmin=1500, nmax=4096, lmin=0, lmax=1024, dtype="bf16"),
        # cached prefixes of a few requests given back for a prompt chunk's attention
        dict(name="read_b8", kind="read", batch=8, heads=4, dim=256, values=True, page=16, lmin=512, lmax=8192, dtype="bf16"),
        # one request's latent rows
        dict(name="read_latent_b1", kind="read", batch=1, heads=1, dim=576, values=False, page=64, lmin=1999, lmax=1999,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between ``lo`` and ``hi``, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(("latent", "latent", "latent", "sample", "sample", "sample", "write", "read"))
        ragged = rng.random() < 0.5
        lmax = _log(rng, 1, 16384)
        lmin = max(0, lmax // rng.choice((1, 2, 8)) - rng.choice((0, 1)))
        page = rng.choice((16, 16, 64, 24))
        if kind == "latent":
            dtype, cache = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("f16", "fp8")))
            case = dict(kind=kind, rank=rng.choice((512, 512, 256)), rope=64, page=page, dtype=dtype, batch=_log(rng, 1, 256),
                        width=rng.choice((1, 2, rng.randint(3, 32))), ragged=ragged, heads=rng.choice((8, 16, 32, 64, 128)),
                        lmin=lmin, lmax=lmax, cache=cache)
        elif kind == "sample":
            chain = rng.random() < 0.4
            case = dict(kind=kind, batch=_log(rng, 1, 256), width=rng.randint(2, 8) if chain else rng.randint(3, 32), chain=chain,
                        ragged=ragged, vocab=rng.choice((151936, 151936, 50257, 32000, rng.randint(300, 5000))),
                        dtype=rng.choice(("bf16", "bf16", "f16", "f32")), probs=rng.choice(("", "", "f32", "bf16")))
        elif kind == "write":
            path = rng.random() < 0.6
            width = rng.randint(2, 32) if path else 0
            nmax = width or _log(rng, 1, 4096)
            heads, dim, values = rng.choice(((4, 256, True), (8, 128, True), (1, 256, True), (1, 576, False), (2, 64, True)))
            case = dict(kind=kind, batch=_log(rng, 1, 256 if path else 16), width=width, path=path, heads=heads, dim=dim,
                        values=values, page=page, nmin=nmax if path else max(1, nmax // 3), nmax=nmax, lmin=min(lmin, 4096),
                        lmax=min(lmax, 4096), dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
        else:
            heads, dim, values = rng.choice(((4, 256, True), (8, 128, True), (1, 256, True), (1, 576, False), (2, 64, True)))
            case = dict(kind=kind, batch=_log(rng, 1, 64), heads=heads, dim=dim, values=values, page=page, lmin=lmin, lmax=lmax,
                        dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
        if _affordable(case):
            return case


def _affordable(c):
    """No more work, and no larger padded arrays, than the largest listed case of its kind."""
    if c["kind"] == "latent":
        padded = c["batch"] * (c["lmax"] + c["width"])
        return work(c)["flops"] <= 1.2e11 and padded <= 128 * 8196 and padded * c["width"] * c["heads"] <= 64 * 8208 * 256
    if c["kind"] == "sample":
        return c["batch"] * c["width"] * c["vocab"] <= 64 * 16 * 151936 * (0.5 if c["probs"] else 1)
    if c["kind"] == "write":
        return c["batch"] * (c["nmax"] + c["page"]) * c["heads"] * c["dim"] <= 4 * 4112 * 1024 and c["batch"] * c["lmax"] <= 1 << 18
    return c["batch"] * c["lmax"] * c["heads"] * c["dim"] <= 8 * 8192 * 1024


# ---- sizes -------------------------------------------------------------------------------------------------------------
def _sizes(c):
    """A request's rows (a tree's nodes) and context (or rows to read), as lists over the batch: the case alone gives
    them, so that every seed's outputs have one shape."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    context = [rng.randint(c["lmin"], c["lmax"]) if "lmin" in c else 0 for _ in range(c["batch"])]
    if c["kind"] == "write":
        return [rng.randint(c["nmin"], c["nmax"]) for _ in context], context
    w = c.get("width", 0)
    return [rng.randint(max(1, w // 2), w) if c.get("ragged") else w for _ in context], context


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
HIT = 0.7  # about the probability that some child of a node is accepted, as the inputs below make it


def _visited(c):
    """Expected nodes on a request's walk: every node at its chance of being reached, over sixteen trees of the rule."""
    total, rng = 0.0, random.Random(1)
    for _ in range(16):
        parents = _parents(rng, c["width"], c["chain"])
        kids = [parents.count(n) for n in range(len(parents))]
        reach = [1.0] * len(parents)
        for r in range(1, len(parents)):
            reach[r] = reach[parents[r]] * HIT / kids[parents[r]]
        total += sum(reach)
    return total / 16


def work(case):
    c = case
    nodes, context = _sizes(c)
    if c["kind"] == "latent":
        dim, eb, rows = c["rank"] + c["rope"], BYTES[c["cache"]], sum(nodes)
        moved = sum(context) * dim * eb + rows * dim * 2 + rows * c["heads"] * (dim + c["rank"]) * 2
        pairs = sum(n * (k + 1) for n, k in zip(nodes, context))  # a row sees the context and itself at least
        return {"bytes": moved, "flops": 2.0 * pairs * c["heads"] * (dim + c["rank"])}
    if c["kind"] == "sample":  # the rows of the nodes on the walk; the draft's row where the walk ends with a rejection
        rows = c["batch"] * _visited(c)
        moved = rows * c["vocab"] * BYTES[c["dtype"]]
        if c["probs"]:
            moved += c["batch"] * (1 - HIT ** (c["width"] - 1)) * c["vocab"] * BYTES[c["probs"]]
        return {"bytes": moved, "flops": rows * c["vocab"] * 4.0}
    if c["kind"] == "write":
        rows = c["batch"] * (1 + max(1, c["width"] // 2)) / 2 if c["path"] else sum(nodes)
        values = rows * c["heads"] * c["dim"] * (2 if c["values"] else 1)
        return {"bytes": values * (BYTES[c["dtype"]] + 1), "flops": values * 2.0}
    values = sum(context) * c["heads"] * c["dim"] * (2 if c["values"] else 1)
    return {"bytes": max(1.0, values * (1 + BYTES[c["dtype"]])), "flops": values}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _parents(rng, n, chain):
    """Parent row of every row of a tree of ``n`` rows, parents first."""
    if chain:
        return [r - 1 for r in range(n)]
    parents, kids, depth = [-1], [0], [0]
    for r in range(1, n):
        p = rng.choice([x for x in range(r) if kids[x] < MAX_CHILDREN and depth[x] < 12])
        parents.append(p)
        kids[p] += 1
        kids.append(0)
        depth.append(depth[p] + 1)
    return parents


def _trees(c, rng):
    """Parents of every request, the first row of each (and the total), and the [batch, W] parent table."""
    w, sizes = c["width"], _sizes(c)[0]
    trees = [_parents(rng, n, c.get("chain", False)) for n in sizes]
    table = np.full((c["batch"], w), -1, dtype=np.int32)
    for b, t in enumerate(trees):
        table[b, : len(t)] = t
    return trees, np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32), table


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


def _power_scale(amax):
    """The least power of two ``s`` with ``amax <= 448 s`` (0 for 0), in fp32."""
    mant, exp = torch.frexp(amax.double() / E4M3_MAX)
    exp = torch.where(mant > 0.5, exp, exp - 1).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(mant), exp), 0.0).float()


def _quantized(x):
    """fp8 pages of ``x`` [blocks, page, heads, dim] and their scales [blocks, heads]."""
    scale = _power_scale(x.abs().amax((1, 3)))
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    return (x * inv[:, None, :, None]).to(torch.float8_e4m3fn), scale


def _cache(gen, dev, blocks, page, heads, dim, kind):
    """Pages of values whose size differs from page to page, and their scales (fp8)."""
    size = 0.25 + 1.5 * torch.rand(blocks, 1, heads, 1, generator=gen, device=dev)
    x = torch.randn(blocks, page, heads, dim, generator=gen, device=dev) * size
    return _quantized(x) if kind == "fp8" else (x.to(DTYPES[kind]), None)


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    rng = random.Random(int(seed) * 7919 + 17)
    gen = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    return {"latent": _prepare_latent, "sample": _prepare_sample, "write": _prepare_write,
            "read": _prepare_read}[c["kind"]](c, rng, gen, dev, on)


def _prepare_latent(c, rng, gen, dev, on):
    trees, starts, _ = _trees(c, rng)
    context = np.array(_sizes(c)[1], dtype=np.int32)
    table, blocks = _pages(rng, context + c["width"], c["page"])
    dim = c["rank"] + c["rope"]
    cache, scale = _cache(gen, dev, blocks, c["page"], 1, dim, c["cache"])
    masks = np.zeros((c["batch"], c["width"]), dtype=np.int64)
    for b, parents in enumerate(trees):
        for r, p in enumerate(parents):
            masks[b, r] = (1 << r) | (int(masks[b, p]) if r else 0)
    tokens, dt = int(starts[-1]), DTYPES[c["dtype"]]
    return SimpleNamespace(
        kind="latent", q=torch.randn(tokens, c["heads"], dim, generator=gen, device=dev).to(dt),
        new=torch.randn(tokens, dim, generator=gen, device=dev).to(dt), cache=cache[:, :, 0],
        cache_scale=None if scale is None else scale[:, 0], table=on(table), context=on(context), starts=on(starts),
        masks=on(masks), scale=(128 + c["rope"]) ** -0.5, width=c["width"], longest=int(context.max()),
        out=torch.empty(tokens, c["heads"], c["rank"], dtype=dt, device=dev))


def _prepare_sample(c, rng, gen, dev, on):
    trees, starts, table = _trees(c, rng)
    rows, vocab = int(starts[-1]), c["vocab"]
    parent = np.concatenate([np.array(t) + starts[b] for b, t in enumerate(trees)])  # row of the parent; a root: before it
    is_child = np.concatenate([np.arange(len(t)) > 0 for t in trees])
    parent, is_child = on(np.where(is_child, parent, 0).astype(np.int64)), on(is_child)
    # a language model's logits: a broad floor, some two dozen likely tokens, and (below) the drafted ones
    floor = 4.2 * math.sqrt(math.log(max(vocab, 2)) / math.log(151936))
    logits = torch.randn(rows, vocab, generator=gen, device=dev) * (0.45 * floor)
    likely = torch.randint(0, vocab, (rows, 24), generator=gen, device=dev)
    base = math.log(vocab)
    logits.scatter_(1, likely, base + 0.6 + 1.5 * torch.randn(rows, 24, generator=gen, device=dev))
    drafted = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
    probs = None
    temperature = 0.7 + 0.3 * torch.rand(c["batch"], generator=gen, device=dev)
    request = torch.repeat_interleave(torch.arange(c["batch"], device=dev), on(np.diff(starts)).long())
    if c["probs"]:
        guess = logits + 0.9 * torch.randn(rows, vocab, generator=gen, device=dev)
        probs = torch.softmax(guess / temperature[request][:, None], -1).to(DTYPES[c["probs"]])
        del guess
        step = 256  # the drafted tokens, drawn from their parents' rows
        for at in range(0, rows, step):
            drafted[at : at + step] = torch.multinomial(probs[parent[at : at + step]].float(), 1, generator=gen)[:, 0]
    else:
        logits[parent[is_child], drafted[is_child]] = base + 4.85 + 0.7 * torch.randn(int(is_child.sum()), generator=gen,
                                                                                  device=dev)
    slots = torch.randperm(c["batch"] + 2, generator=gen, device=dev)[: c["batch"]].to(torch.int32)
    parents = torch.full((c["batch"] + 2, c["width"]), -1, dtype=torch.int32, device=dev)
    parents[slots.long()] = on(table)
    store = SimpleNamespace(width=c["width"], parents=parents, path=torch.zeros_like(parents),
                            path_len=torch.ones(c["batch"] + 2, dtype=torch.int32, device=dev))
    return SimpleNamespace(
        kind="sample", logits=logits.to(DTYPES[c["dtype"]]), drafted=drafted, starts=on(starts), slots=slots, store=store,
        coins=torch.rand(rows, generator=gen, device=dev), final=torch.rand(c["batch"], generator=gen, device=dev),
        temperature=temperature, probs=probs)


def _prepare_write(c, rng, gen, dev, on):
    counts, context = (np.array(x, dtype=np.int32) for x in _sizes(c))
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    table, blocks = _pages(rng, context + counts, c["page"])
    tokens, dt = int(starts[-1]), DTYPES[c["dtype"]]
    key_cache, k_scale = _cache(gen, dev, blocks, c["page"], c["heads"], c["dim"], "fp8")
    value_cache, v_scale = _cache(gen, dev, blocks, c["page"], c["heads"], c["dim"], "fp8") if c["values"] else (None, None)
    path = path_len = slots = None
    if c["path"]:
        slots = torch.randperm(c["batch"] + 2, generator=gen, device=dev)[: c["batch"]].to(torch.int32)
        paths, lens = np.zeros((c["batch"] + 2, c["width"]), dtype=np.int32), np.ones(c["batch"] + 2, dtype=np.int32)
        for b in range(c["batch"] + 2):
            n = rng.randint(1, max(1, c["width"] // 2))
            paths[b, :n] = sorted([0] + rng.sample(range(1, c["width"]), n - 1))
            lens[b] = n
        path, path_len = on(paths), on(lens)
    rows = lambda: (torch.randn(tokens, c["heads"], c["dim"], generator=gen, device=dev) * (  # noqa: E731
        0.25 + 2.0 * torch.rand(tokens, c["heads"], 1, generator=gen, device=dev))).to(dt)
    return SimpleNamespace(kind="write", key=rows(), value=rows() if c["values"] else None, key_cache=key_cache,
                           value_cache=value_cache, k_scale=k_scale, v_scale=v_scale, table=on(table), context=on(context),
                           starts=on(starts), most=int(counts.max()), slots=slots, path=path, path_len=path_len)


def _prepare_read(c, rng, gen, dev, on):
    lens = np.array(_sizes(c)[1], dtype=np.int32)
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    table, blocks = _pages(rng, lens, c["page"])
    key_cache, k_scale = _cache(gen, dev, blocks, c["page"], c["heads"], c["dim"], "fp8")
    value_cache, v_scale = _cache(gen, dev, blocks, c["page"], c["heads"], c["dim"], "fp8") if c["values"] else (None, None)
    empty = lambda: torch.empty(int(starts[-1]), c["heads"], c["dim"], dtype=DTYPES[c["dtype"]], device=dev)  # noqa: E731
    return SimpleNamespace(kind="read", key_cache=key_cache, value_cache=value_cache, k_scale=k_scale, v_scale=v_scale,
                           table=on(table), starts=on(starts), most=int(lens.max()), key=empty(),
                           value=empty() if c["values"] else None)


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        return _call(s)
    return {"latent": _latent, "sample": _sample, "write": _write, "read": _read}[s.kind](s)


def _call(s):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    if s.kind == "latent":
        from eagle_harness.vllm.latent_attention import latent_verify_attention

        return latent_verify_attention(s.q, s.new, s.cache, s.table, s.context, s.starts, s.masks, s.scale, s.out,
                                       max_query_len=s.width, latent_scale=s.cache_scale)
    if s.kind == "sample":
        from eagle_harness.vllm.tree_accept import sample_tree

        sampled, count = sample_tree(s.logits, s.drafted, s.starts, s.slots, s.store.parents, s.store, s.coins, s.final,
                                     s.temperature, draft_probs=s.probs)
        return sampled, count, s.store.path, s.store.path_len
    if s.kind == "write":
        from eagle_harness.vllm.kv_pages import write_kv_pages

        write_kv_pages(s.key, s.value, s.key_cache, s.value_cache, s.k_scale, s.v_scale, s.table, s.context, s.starts,
                       max_query_len=s.most, idx_mapping=s.slots, path=s.path, path_len=s.path_len)
        return s.key_cache, s.k_scale, s.value_cache, s.v_scale
    from eagle_harness.vllm.kv_pages import read_kv_pages

    read_kv_pages(s.key_cache, s.value_cache, s.k_scale, s.v_scale, s.table, s.starts, s.key, s.value, max_len=s.most)
    return s.key, s.value


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _of_rows(starts, total, dev):
    """Request and local index of every one of ``total`` rows, ``starts`` the first row of each request."""
    rows = torch.arange(total, device=dev)
    request = torch.searchsorted(starts.long(), rows, right=True) - 1
    return request, rows - starts.long()[request]


def _latent(s):
    rank, dim, heads = s.out.shape[-1], s.q.shape[-1], s.q.shape[1]
    page, dev = s.cache.shape[1], s.q.device
    request, local = _of_rows(s.starts, s.q.shape[0], dev)
    counts = (s.starts[1:] - s.starts[:-1])[:, None]
    rows = torch.arange(s.width, device=dev)[None]
    token = (s.starts[:-1, None] + rows).clamp(max=s.q.shape[0] - 1).long()  # [R, W]; rows past a request's are dropped
    at = torch.arange(s.longest, device=dev)
    blocks = s.table[:, at // page].long()  # [R, L]
    keys = s.cache[blocks, at % page].float() if s.cache_scale is None else \
        s.cache.float()[blocks, at % page] * s.cache_scale[blocks][..., None]
    keys = torch.cat([keys, s.new[token].float()], 1)  # [R, L + W, dim]
    bits = (s.masks[:, :, None] >> rows[None]) & 1
    seen = torch.cat([(at[None] < s.context[:, None])[:, None].expand(-1, s.width, -1),
                      (bits == 1) & (rows < counts)[:, None]], 2)
    q = s.q[token].float().reshape(token.shape[0], s.width * heads, dim)
    score = torch.matmul(q, keys.transpose(1, 2)).view(token.shape[0], s.width, heads, -1) * s.scale
    score = torch.where(seen[:, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    got = torch.matmul(weight.flatten(1, 2), keys[..., :rank]).view(token.shape[0], s.width, heads, rank)
    got = torch.where(total > 0, got / total, 0.0)
    return s.out.copy_(got[request, local])


def _sample(s):
    """Every row's outcome as if the walk came there, then the rows whose whole path was taken."""
    dev, width, (total, vocab) = s.logits.device, s.store.width, s.logits.shape
    requests, slot = s.starts.shape[0] - 1, s.slots.long()
    request, local = _of_rows(s.starts, total, dev)
    rows, child = torch.arange(total, device=dev), local > 0
    first = rows - local
    parent = first + s.store.parents[slot].long()[request, local].clamp(min=0)
    p = s.logits.double()
    p = torch.exp((p - p.amax(1, keepdim=True)) / s.temperature.double()[request][:, None])
    p = p / p.sum(1, keepdim=True)
    # the order of a row among its siblings, and the children of every row by that order
    same = (parent[:, None] == parent[None]) & child[:, None] & child[None] & (rows[None] < rows[:, None])
    spot = torch.where(child, parent * MAX_CHILDREN + same.sum(1), total * MAX_CHILDREN)
    kids = torch.full((total * MAX_CHILDREN + 1,), -1, dtype=torch.int64, device=dev)
    kids = kids.scatter(0, spot, rows)[:-1].view(total, MAX_CHILDREN)
    taken = torch.full((total,), -1, dtype=torch.int64, device=dev)
    spent = torch.zeros(total, dtype=torch.float64, device=dev)
    left, mass = p, torch.ones(total, dtype=torch.float64, device=dev)
    q = None if s.probs is None else s.probs.double()
    for k in range(MAX_CHILDREN):
        kid = kids[:, k]
        trying = (kid >= 0) & (taken < 0)
        token = s.drafted[kid.clamp(min=0)][:, None]
        chance = left.gather(1, token)[:, 0]
        drawn = 1.0 if q is None else q.gather(1, token)[:, 0]
        good = trying & (s.coins[kid.clamp(min=0)].double() * drawn * mass < chance)
        taken = torch.where(good, kid, taken)
        lost = trying & ~good
        if q is None:
            left = left.scatter(1, token, torch.where(lost, 0.0, chance)[:, None])
        else:
            spent = spent + torch.where(lost, mass, 0.0)
            left = torch.clamp(p - spent[:, None] * q, min=0.0)
        mass = left.sum(1)
    left = torch.where((mass > 0)[:, None], left, p)
    # reached: every row of the path from the root is the one its parent chose
    chosen = (taken[parent] == rows) | ~child
    reached, at = chosen, rows
    for _ in range(min(width, 13)):  # a tree is at most 12 deep
        at = torch.where(child[at], parent[at], at)
        reached = reached & chosen[at]
    before = torch.cumsum(reached.long(), 0) - reached.long()
    place = before - before[first]
    count = torch.zeros(requests, dtype=torch.int32, device=dev).index_add_(0, request, reached.int())
    spare = requests * width  # one entry past the tables takes what is not kept
    path = torch.zeros(spare + 1, dtype=torch.int64, device=dev)
    path = path.scatter(0, torch.where(reached, request * width + place, spare), local)[:-1].view(requests, width)
    end = torch.zeros(requests + 1, dtype=torch.int64, device=dev)
    end = end.scatter(0, torch.where(reached & (taken < 0), request, requests), rows)[:-1]
    running = torch.cumsum(left[end], 1)
    final = torch.searchsorted(running, s.final.double()[:, None] * running[:, -1:], right=True).clamp(max=vocab - 1)
    sampled = torch.full((spare + 1,), -1, dtype=torch.int64, device=dev)
    sampled = sampled.scatter(0, torch.where(reached & child, request * width + place - 1, spare), s.drafted)
    sampled = sampled[:-1].view(requests, width).scatter(1, count.long()[:, None] - 1, final)
    live = torch.arange(width, device=dev)[None] < count[:, None]
    s.store.path[slot] = torch.where(live, path.int(), s.store.path[slot])
    s.store.path_len[slot] = count
    return sampled, count, s.store.path, s.store.path_len


def _write(s):
    """Every request writes a row at least; entries past a request's rows repeat its first row's write."""
    dev, page = s.key.device, s.key_cache.shape[1]
    j, width = torch.arange(s.most, device=dev)[None], s.starts.shape[0] - 1
    count = (s.starts[1:] - s.starts[:-1] if s.path is None else s.path_len[s.slots.long()]).long()[:, None]
    j = torch.where(j < count, j, 0)
    src = j if s.path is None else s.path[s.slots.long()].long().gather(1, j)
    pos = s.context.long()[:, None] + j
    row, block, at = s.starts.long()[:-1, None] + src, s.table.gather(1, pos // page).long(), pos % page
    first = s.context.long()[:, None] // page
    pages = (s.most + page - 1) // page + 1
    index = torch.arange(pages, device=dev)[None]
    index = torch.where((first + index) * page < s.context[:, None] + count, index, 0)  # the pages that rows go to
    blocks = s.table.gather(1, first + index).long()
    kept = s.context[:, None] % page  # rows of the first page that stay
    lead = torch.arange(page, device=dev)[None].expand(width, -1)
    for x, cache, scale in ((s.key, s.key_cache, s.k_scale), (s.value, s.value_cache, s.v_scale)):
        if x is None:
            continue
        raw, rows = cache.view(torch.uint8), x[row].float()  # [R, most, heads, dim]
        size = torch.where(torch.isfinite(rows), rows.abs(), 0.0).amax(-1)
        most = torch.zeros(width, pages, x.shape[1], device=dev)
        most.scatter_reduce_(1, (pos // page - first)[..., None].expand_as(size), size, "amax")
        most = most.gather(1, index[..., None].expand_as(most))
        old = torch.where(((index == 0) & (kept > 0))[..., None], scale[blocks], 0.0)
        new = torch.maximum(old, _power_scale(most))
        held = raw[blocks[:, 0]]  # the first page's earlier rows at its new scale
        ratio = torch.where(new[:, 0] > 0, old[:, 0] / new[:, 0], 0.0)
        again = (held.view(cache.dtype).float() * ratio[:, None, :, None]).to(cache.dtype).view(torch.uint8)
        raw[blocks[:, :1].expand_as(lead), lead] = torch.where((lead < kept)[..., None, None], again, held)
        scale[blocks] = new
        factor = scale[block]
        value = rows * torch.where(factor > 0, 1.0 / factor, 0.0)[..., None]
        raw[block, at] = value.clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype).view(torch.uint8)
    return s.key_cache, s.k_scale, s.value_cache, s.v_scale


def _read(s):
    page, out = s.key_cache.shape[1], s.key
    request, at = _of_rows(s.starts, out.shape[0], out.device)
    block = s.table[request, at // page].long()
    for out, cache, scale in ((s.key, s.key_cache, s.k_scale), (s.value, s.value_cache, s.v_scale)):
        if out is not None:
            raw = cache.view(torch.uint8)[block, at % page]
            out.copy_(raw.view(cache.dtype).float() * scale[block][..., None])
    return s.key, s.value


# ---- the same in 64 bits, request by request -----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"latent": _latent64, "sample": lambda s: None, "write": _write64, "read": _read64}[s.kind](s)


def _rows64(cache, scale, table, positions):
    """Rows of one request's positions in 64 bits; ``table`` its row of the block table."""
    page = cache.shape[1]
    block = table[positions // page].long()
    rows = cache[block, positions % page].double() if cache.dtype != torch.float8_e4m3fn else \
        cache.view(torch.uint8)[block, positions % page].view(cache.dtype).double()
    if scale is not None:
        factor = scale[block].double()
        rows = rows * factor.reshape(factor.shape + (1,) * (rows.dim() - factor.dim()))
    return rows


def _latent64(s):
    rank = s.out.shape[-1]
    got = torch.zeros(s.out.shape, dtype=torch.float64, device=s.out.device)
    starts, context, masks = s.starts.tolist(), s.context.tolist(), s.masks.tolist()
    for b, length in enumerate(context):
        held = _rows64(s.cache, s.cache_scale, s.table[b], torch.arange(length, device=s.out.device))
        for r in range(starts[b + 1] - starts[b]):
            chosen = [starts[b] + k for k in range(starts[b + 1] - starts[b]) if masks[b][r] >> k & 1]
            keys = torch.cat([held, s.new[chosen].double()])
            if keys.shape[0]:
                weight = torch.softmax(s.q[starts[b] + r].double() @ keys.t() * s.scale, -1)
                got[starts[b] + r] = weight @ keys[:, :rank]
    return got


def _write64(s):
    page = s.key_cache.shape[1]
    starts, context, table = s.starts.tolist(), s.context.tolist(), s.table.tolist()
    outs = []
    for x, cache, scale in ((s.key, s.key_cache, s.k_scale), (s.value, s.value_cache, s.v_scale)):
        if x is None:
            outs += [None, None]
            continue
        held, factor, rows = cache.double().cpu().numpy(), scale.double().cpu().numpy(), x.double().cpu().numpy()
        for b, length in enumerate(context):
            if s.path is None:
                source = list(range(starts[b], starts[b + 1]))
            else:
                slot = int(s.slots[b])
                source = [starts[b] + r for r in s.path[slot, : int(s.path_len[slot])].tolist()]
            done = 0
            while done < len(source):
                at, lead = table[b][(length + done) // page], (length + done) % page
                part = rows[source[done : done + page - lead]]
                most = np.abs(part).max((0, 2))
                need = np.where(most > 0, 2.0 ** np.ceil(np.log2(np.maximum(most, 1e-300) / E4M3_MAX)), 0.0)
                now = np.maximum(need, factor[at]) if lead else need
                safe = np.where(now > 0, now, 1.0)[:, None]
                if lead:
                    held[at, :lead] *= factor[at][:, None] / safe
                held[at, lead : lead + len(part)] = part / safe
                factor[at] = now
                done += len(part)
        outs += [torch.from_numpy(held), torch.from_numpy(factor)]
    return tuple(outs)


def _read64(s):
    starts = s.starts.tolist()
    outs = []
    for out, cache, scale in ((s.key, s.key_cache, s.k_scale), (s.value, s.value_cache, s.v_scale)):
        if out is None:
            outs.append(None)
            continue
        parts = [_rows64(cache, scale, s.table[b], torch.arange(starts[b + 1] - starts[b], device=cache.device))
                 for b in range(len(starts) - 1)]
        outs.append(torch.cat(parts))
    return tuple(outs)
