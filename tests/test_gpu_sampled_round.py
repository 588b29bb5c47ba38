"""A sampled verify round over quantized caches as a server runs it: prompts written into fp8 pages, tree attention over grouped
and over latent heads, the sampled walk, the accepted rows written behind the context, the next round on what they left, and the
pages read back. Every step against its oracle on what the step was given; then the round captured once and replayed."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import attention as oa
from oracle import kv_pages as okv
from oracle import latent as olat
from oracle import sampling as osm
from test_gpu_attention import _close
from test_gpu_kv_pages import same
from workloads import seeded_tree, tree_masks

pytestmark = pytest.mark.gpu

BF16, F32, FP8, I32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int32
HEADS, KV, D, RANK, ROPE, PAGE, WIDTH, VOCAB, SLOTS = 16, 4, 128, 512, 64, 16, 8, 1000, 6
CONTEXTS, SIZES, ROUNDS = [37, 0, 112, 64], [8, 5, 1, 8], 3
DIM, TOKENS, REQS = RANK + ROPE, sum(SIZES), len(SIZES)


def server(dev, seed):
    """What stays on the device between rounds: empty pages, the tables, a head of random weights."""
    gen = torch.Generator().manual_seed(seed)
    most = -(-(max(CONTEXTS) + ROUNDS * WIDTH) // PAGE) + 1
    blocks = REQS * most + 2
    table = torch.randperm(blocks, generator=gen)[: REQS * most].view(REQS, most).to(I32)

    def pages(heads, dim):
        return torch.zeros(blocks, PAGE, heads, dim).to(FP8).to(dev), torch.zeros(blocks, heads, device=dev)

    k, ks = pages(KV, D)
    v, vs = pages(KV, D)
    lat, ls = pages(1, DIM)
    return SimpleNamespace(
        k=k, ks=ks, v=v, vs=vs, lat=lat, ls=ls, table=table.to(dev), context=torch.tensor(CONTEXTS, dtype=I32, device=dev),
        starts=torch.tensor([0, *np.cumsum(SIZES)], dtype=I32, device=dev),
        slots=torch.tensor([4, 0, 5, 2], dtype=I32, device=dev),
        store=SimpleNamespace(width=WIDTH, path=torch.zeros(SLOTS, WIDTH, dtype=I32, device=dev),
                              path_len=torch.zeros(SLOTS, dtype=I32, device=dev)),
        head=(torch.randn(HEADS * D, VOCAB, generator=gen) * 0.1).to(dev),
        latent_head=(torch.randn(HEADS * RANK, VOCAB, generator=gen) * 0.05).to(dev),
        out=torch.zeros(TOKENS, HEADS, D, dtype=BF16, device=dev),
        latent_out=torch.zeros(TOKENS, HEADS, RANK, dtype=BF16, device=dev))


def drafts(dev, seed):
    """A round's inputs: trees, rows and coins."""
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    masks = torch.zeros(REQS, WIDTH, dtype=torch.int64)
    parents = torch.full((SLOTS, WIDTH), -1, dtype=I32)
    for b, n in enumerate(SIZES):
        tree = seeded_tree(rng, n)
        masks[b, :n] = torch.tensor(tree_masks(tree))
        parents[[4, 0, 5, 2][b], :n] = torch.tensor(tree, dtype=I32)
    x = dict(
        q=torch.randn(TOKENS, HEADS, D, generator=gen).to(BF16), k=torch.randn(TOKENS, KV, D, generator=gen).to(BF16),
        v=torch.randn(TOKENS, KV, D, generator=gen).to(BF16), lq=torch.randn(TOKENS, HEADS, DIM, generator=gen).to(BF16),
        lat=torch.randn(TOKENS, DIM, generator=gen).to(BF16), masks=masks, parents=parents,
        drafted=torch.randint(0, VOCAB, (TOKENS,), generator=gen), coins=torch.rand(TOKENS, generator=gen) * 0.002,
        final=torch.rand(REQS, generator=gen), temperature=torch.tensor([1.0, 0.5, 0.0, 1.5]))
    return SimpleNamespace(**{k: t.to(dev) for k, t in x.items()})


def fill(s, seed):
    """The prompts, written into the pages from their start."""
    from eagle_harness.vllm.kv_pages import write_kv_pages

    gen = torch.Generator().manual_seed(seed)
    dev, n = s.table.device, sum(CONTEXTS)
    rows = [torch.randn(n, KV, D, generator=gen).to(BF16).to(dev), torch.randn(n, KV, D, generator=gen).to(BF16).to(dev),
            torch.randn(n, 1, DIM, generator=gen).to(BF16).to(dev)]
    starts = torch.tensor([0, *np.cumsum(CONTEXTS)], dtype=I32, device=dev)
    none = torch.zeros_like(s.context)
    write_kv_pages(rows[0], rows[1], s.k, s.v, s.ks, s.vs, s.table, none, starts, max_query_len=max(CONTEXTS))
    write_kv_pages(rows[2], None, s.lat, None, s.ls, None, s.table, none, starts, max_query_len=max(CONTEXTS))
    return rows, starts


def forward(s, x):
    from eagle_harness.vllm.latent_attention import latent_verify_attention
    from eagle_harness.vllm.verify_attention import verify_attention

    verify_attention(x.q, x.k, x.v, s.k, s.v, s.table, s.context, s.starts, x.masks, D ** -0.5, s.out, max_query_len=WIDTH,
                     k_scale=s.ks, v_scale=s.vs)
    latent_verify_attention(x.lq, x.lat, s.lat[:, :, 0], s.table, s.context, s.starts, x.masks, DIM ** -0.5, s.latent_out,
                            max_query_len=WIDTH, latent_scale=s.ls)
    return s.out.float().flatten(1) @ s.head + s.latent_out.float().flatten(1) @ s.latent_head


def walk(s, x, logits):
    from eagle_harness.vllm.tree_accept import sample_tree

    return sample_tree(logits, x.drafted, s.starts, s.slots, x.parents, s.store, x.coins, x.final, x.temperature)


def commit(s, x):
    from eagle_harness.vllm.kv_pages import write_kv_pages

    paths = dict(max_query_len=WIDTH, idx_mapping=s.slots, path=s.store.path, path_len=s.store.path_len)
    write_kv_pages(x.k, x.v, s.k, s.v, s.ks, s.vs, s.table, s.context, s.starts, **paths)
    write_kv_pages(x.lat[:, None], None, s.lat, None, s.ls, None, s.table, s.context, s.starts, **paths)
    s.context.add_(s.store.path_len[s.slots.long()])


def host(*tensors):
    return [t.detach().cpu().clone() for t in tensors]


def test_rounds_match_the_oracles(dev):
    announce("sampled rounds over fp8 pages")
    s = server(dev, 1)
    want = dict(zip(("k", "ks", "v", "vs", "lat", "ls"), host(s.k, s.ks, s.v, s.vs, s.lat, s.ls)))
    table, starts, slots = host(s.table, s.starts, s.slots)

    def pages_match():
        for name in ("k", "v", "lat"):
            assert same(getattr(s, name), want[name]), name
        for name in ("ks", "vs", "ls"):
            assert torch.equal(getattr(s, name).cpu(), want[name]), name

    rows, prompt_starts = fill(s, 2)
    for r, cache, scale in ((rows[0], "k", "ks"), (rows[1], "v", "vs"), (rows[2], "lat", "ls")):
        okv.write_pages(r.cpu(), want[cache], want[scale], table, [0] * REQS, prompt_starts.cpu())
    pages_match()
    accepted = 0
    for round_ in range(ROUNDS):
        x = drafts(dev, 10 + round_)
        h = SimpleNamespace(**dict(zip(vars(x), host(*vars(x).values()))))
        context, = host(s.context)
        logits = forward(s, x)
        _close(s.out.cpu(), oa.verify_attention(h.q, h.k, h.v, want["k"], want["v"], table, context, starts, h.masks, D ** -0.5,
                                                torch.zeros(TOKENS, HEADS, D, dtype=BF16), max_query_len=WIDTH,
                                                k_scale=want["ks"], v_scale=want["vs"]))
        lat, bound = olat.latent_attention(h.lq, h.lat, want["lat"][:, :, 0], table, context, starts, h.masks, DIM ** -0.5, RANK,
                                           want["ls"][:, 0])
        assert bool(((s.latent_out.cpu().double() - lat).abs() <= bound).all())

        path, path_len = host(s.store.path, s.store.path_len)
        sampled, count = walk(s, x, logits)
        tokens, num = osm.sample_tree(logits.cpu(), h.drafted, starts, slots, h.parents, h.coins, h.final, h.temperature, path,
                                      path_len, WIDTH)
        assert count.cpu().tolist() == num.tolist() and sampled.cpu().tolist() == tokens.tolist()
        assert s.store.path.cpu().tolist() == path.tolist() and s.store.path_len.cpu().tolist() == path_len.tolist()
        accepted += int(num.sum()) - REQS

        commit(s, x)
        for r, cache, scale in ((h.k, "k", "ks"), (h.v, "v", "vs"), (h.lat[:, None], "lat", "ls")):
            okv.write_pages(r, want[cache], want[scale], table, context, starts, path=path, path_len=path_len, slots=slots)
        pages_match()
        assert s.context.cpu().tolist() == (context + path_len[slots.long()]).tolist()
    assert accepted > 0  # rows behind the root have been committed

    from eagle_harness.vllm.kv_pages import read_kv_pages

    lengths = [int(c) for c in s.context.cpu()]
    ends = torch.tensor([0, *np.cumsum(lengths)], dtype=I32, device=dev)
    k, v = (torch.zeros(sum(lengths), KV, D, dtype=BF16, device=dev) for _ in range(2))
    lat = torch.zeros(sum(lengths), 1, DIM, dtype=BF16, device=dev)
    read_kv_pages(s.k, s.v, s.ks, s.vs, s.table, ends, k, v, max_len=max(lengths))
    read_kv_pages(s.lat, None, s.ls, None, s.table, ends, lat, None, max_len=max(lengths))
    for got, cache, scale in ((k, "k", "ks"), (v, "v", "vs"), (lat, "lat", "ls")):
        assert torch.equal(got.cpu(), okv.read_pages(want[cache], want[scale], table, ends.cpu()).to(BF16))


def test_a_captured_round_replays(dev):
    """The round as one graph: every replay moves the caches, the contexts and the paths on as the eager round does."""
    announce("a sampled round captured")
    eager, held = server(dev, 3), server(dev, 3)
    fill(eager, 4)
    fill(held, 4)
    x = drafts(dev, 30)
    state = {n: t.clone() for n, t in vars(held).items() if isinstance(t, torch.Tensor)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # libraries set up outside the capture
        walk(held, x, forward(held, x))
        commit(held, x)
    torch.cuda.current_stream().wait_stream(side)
    for n, t in state.items():
        getattr(held, n).copy_(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampled, count = walk(held, x, forward(held, x))
        commit(held, x)
    for round_ in range(ROUNDS):
        new = drafts(dev, 31 + round_)
        for n, t in vars(new).items():
            getattr(x, n).copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = walk(eager, new, forward(eager, new))
        commit(eager, new)
        torch.cuda.synchronize()
        assert torch.equal(sampled, want[0]) and torch.equal(count, want[1])
        for n in ("k", "v", "lat"):
            assert same(getattr(held, n), getattr(eager, n)), n
        for n in ("ks", "vs", "ls", "context", "out", "latent_out"):
            assert torch.equal(getattr(held, n), getattr(eager, n)), n
        assert torch.equal(held.store.path_len, eager.store.path_len)
