"""Tree acceptance by sampling on the GPU against the 64-bit oracle, token for token: every type, odd vocabularies and row
strides, trees and chains, masked and degenerate rows, coins at their ends, other streams and replayed graphs."""

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import sampling as osm
from workloads import seeded_tree

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Store:
    def __init__(self, slots, width, dev):
        self.width = width
        self.path = torch.full((slots, width), -7, dtype=torch.int32, device=dev)
        self.path_len = torch.full((slots,), -7, dtype=torch.int32, device=dev)


def inputs(sizes, width, vocab, dtype, probs, seed, chain=False):
    """A batch on the host: peaked rows, drafted tokens that are often accepted, some siblings alike."""
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    rows, reqs = sum(sizes), len(sizes)
    logits = torch.randn(rows, vocab, generator=gen) * 2
    drafted = torch.zeros(rows, dtype=torch.int64)
    slots = torch.randperm(reqs + 3, generator=gen)[:reqs].to(torch.int32)
    parents = torch.full((reqs + 3, width), -1, dtype=torch.int32)
    cu = torch.tensor([0, *np.cumsum(sizes)], dtype=torch.int32)
    temperature = 0.4 + torch.rand(reqs, generator=gen)
    q = None
    if probs is not None:
        q = torch.softmax(logits + 0.7 * torch.randn(rows, vocab, generator=gen), -1).to(probs)
    for b, n in enumerate(sizes):
        tree = ([r - 1 for r in range(n)] if chain else seeded_tree(rng, n)) if n else []
        m = min(n, width)
        parents[slots[b], :m] = torch.tensor(tree[:m], dtype=torch.int32)
        for r in range(1, n):
            n0 = int(cu[b]) + tree[r]
            if q is not None:
                drafted[cu[b] + r] = int(torch.multinomial(q[n0].float(), 1, generator=gen)[0])
            else:
                token = int(torch.randint(0, vocab, (1,), generator=gen)[0])
                if r % 3 == 0 and r > 1:
                    token = int(drafted[cu[b] + r - 1])  # now and then a sibling's token again
                drafted[cu[b] + r] = token
                logits[n0, token] = 5.0 + 2.0 * float(torch.rand(1, generator=gen)[0]) + np.log(vocab)
    return dict(logits=logits.to(dtype), drafted=drafted, cu=cu, slots=slots, parents=parents,
                coins=torch.rand(rows, generator=gen), final=torch.rand(reqs, generator=gen), temperature=temperature, q=q,
                width=width)


def launch(x, dev, logits=None, q=None):
    from eagle_harness.vllm.tree_accept import sample_tree

    store = Store(x["parents"].shape[0], x["width"], dev)
    probs = x["q"].to(dev) if q is None and x["q"] is not None else q
    sampled, count = sample_tree(x["logits"].to(dev) if logits is None else logits, x["drafted"].to(dev), x["cu"].to(dev),
                                 x["slots"].to(dev), x["parents"].to(dev), store, x["coins"].to(dev), x["final"].to(dev),
                                 x["temperature"].to(dev), draft_probs=probs)
    return sampled, count, store


def expect(x):
    path = torch.full(x["parents"][:, : x["width"]].shape, -7, dtype=torch.int32)
    path_len = torch.full((x["parents"].shape[0],), -7, dtype=torch.int32)
    sampled, count = osm.sample_tree(x["logits"], x["drafted"], x["cu"], x["slots"], x["parents"], x["coins"], x["final"],
                                     x["temperature"], path, path_len, x["width"], x["q"])
    return sampled, count, path, path_len


def check(x, got):
    sampled, count, store = got
    want, num, path, path_len = expect(x)
    assert count.cpu().tolist() == num.tolist()
    assert sampled.cpu().tolist() == want.tolist()
    assert store.path_len.cpu().tolist() == path_len.tolist()
    assert store.path.cpu().tolist() == path.tolist()


@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 513, 1001, 4096, 9000])
@pytest.mark.parametrize("dtype,probs", [(BF16, None), (F16, None), (F32, None), (BF16, F32), (BF16, BF16), (F16, F16),
                                         (F32, F32), (F32, BF16)])
def test_walks_match_the_oracle(dev, vocab, dtype, probs):
    announce(f"sample tree vocab {vocab} {dtype} probs {probs}")
    x = inputs([16, 1, 9, 0, 12, 2, 16], 16, vocab, dtype, probs, seed=vocab)
    check(x, launch(x, dev))


@pytest.mark.parametrize("dtype,probs,vocab", [(BF16, None, 151936), (F32, F32, 50257), (BF16, F32, 151936), (F16, None, 50257)])
def test_full_vocabularies(dev, dtype, probs, vocab):
    announce(f"sample tree vocab {vocab} {dtype} probs {probs}")
    x = inputs([8, 5, 6], 8, vocab, dtype, probs, seed=3, chain=probs is not None)
    check(x, launch(x, dev))


@pytest.mark.parametrize("width,sizes", [(1, [1, 1]), (2, [2, 1]), (5, [9, 5, 3]), (64, [64, 40, 17])])
@pytest.mark.parametrize("probs", [None, F32])
def test_widths(dev, width, sizes, probs):
    announce(f"sample tree width {width} probs {probs}")
    x = inputs(sizes, width, 300, F32, probs, seed=width)
    check(x, launch(x, dev))


@pytest.mark.parametrize("requests", [1, 3, 40, 300])
def test_batches(dev, requests):
    announce(f"sample tree requests {requests}")
    x = inputs([1 + (5 * b) % 7 for b in range(requests)], 8, 700, BF16, None if requests % 2 else F32, seed=requests)
    check(x, launch(x, dev))


@pytest.mark.parametrize("probs", [None, F32])
def test_coins_and_temperatures_at_their_ends(dev, probs):
    announce(f"sample tree ends probs {probs}")
    x = inputs([8] * 8, 8, 200, F32, probs, seed=5)
    below_one = float(np.nextafter(np.float32(1), np.float32(0)))
    x["coins"][:24] = 0.0
    x["coins"][24:40] = below_one
    x["coins"][40:44] = float("nan")
    x["final"][:5] = torch.tensor([0.0, below_one, 1.0, float("nan"), 0.5])
    x["temperature"] = torch.tensor([0.0, 1e-3, 1.0, 1.0, float("inf"), -1.0, 1.0, 0.01])
    x["coins"][16:24] = below_one
    check(x, launch(x, dev))


@pytest.mark.parametrize("probs", [None, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_and_degenerate_rows(dev, dtype, probs):
    announce(f"sample tree degenerate {dtype} probs {probs}")
    x = inputs([6] * 6, 6, 90, dtype, probs, seed=6)
    inf = float("inf")
    x["logits"][0, 30:] = -inf  # tokens that may not be drawn
    x["logits"][6] = -inf       # a row of none
    x["logits"][12, 40] = float("nan")
    x["logits"][18, 5] = x["logits"][18, 50] = inf
    x["logits"][24] = -inf
    x["logits"][24, 77] = -3.0  # one token is left
    x["logits"][30] = torch.finfo(dtype).min  # masked by the lowest value instead
    x["logits"][30, 3] = 1.0
    x["drafted"][1], x["drafted"][2] = -1, 90  # no tokens of the vocabulary
    if probs is not None:
        x["q"][1] = float("nan")
        x["q"][2] = 0.0
        x["q"][25] = 2.0
    check(x, launch(x, dev))


def test_a_residual_of_nothing_falls_back_to_the_targets(dev):
    """Draft probabilities above the target's everywhere (no distribution): after a rejection nothing is left of p."""
    announce("sample tree nothing left")
    x = inputs([3, 3], 3, 50, F32, F32, seed=8, chain=True)
    x["q"][:] = 1.0
    x["coins"][:] = 0.999
    check(x, launch(x, dev))


@pytest.mark.parametrize("dtype,probs", [(BF16, None), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("offset,stride", [(0, 1000), (3, 1007), (1, 1001), (8, 1008)])
def test_strides_and_alignment(dev, dtype, probs, offset, stride):
    announce(f"sample tree {dtype} probs {probs} offset {offset} stride {stride}")
    x = inputs([7, 4], 8, 997, dtype, probs, seed=stride)
    rows = x["logits"].shape[0]
    held = torch.full((rows * stride + 16,), float("inf"), dtype=dtype, device=dev)  # what lies around must not count
    logits = held[offset : offset + rows * stride].view(rows, stride)[:, :997]
    logits.copy_(x["logits"])
    q = None
    if probs is not None:
        q = torch.full((rows, 1003), float("nan"), dtype=probs, device=dev)[:, 2:999]
        q.copy_(x["q"])
    check(x, launch(x, dev, logits, q))


def test_wide_tables_and_longer_parents(dev):
    announce("sample tree int64 tables")
    x = inputs([5, 6, 3], 6, 300, F32, None, seed=12)
    x["cu"], x["slots"], x["drafted"] = x["cu"].long(), x["slots"].long(), x["drafted"].int()
    x["parents"] = torch.cat([x["parents"].long(), torch.full((6, 2), 9)], 1)
    check(x, launch(x, dev))


def test_rows_and_slots_out_of_range_are_skipped(dev):
    """A request whose rows lie outside the logits, or whose slot outside the store: nothing sampled, nothing else touched."""
    announce("sample tree out of range")
    x = inputs([4, 4, 4], 4, 100, F32, None, seed=13)
    whole = launch(x, dev)
    x2 = dict(x, cu=torch.tensor([0, 4, 8, 99], dtype=torch.int32))
    sampled, count, store = launch(x2, dev)
    assert count.cpu().tolist()[:2] == whole[1].cpu().tolist()[:2] and int(count[2]) == 0
    assert sampled[2].cpu().tolist() == [-1] * 4 and torch.equal(sampled[:2], whole[0][:2])
    x3 = dict(x, slots=torch.tensor([int(x["slots"][0]), 1000, -5], dtype=torch.int32))
    sampled, count, store = launch(x3, dev)
    assert count.cpu().tolist()[1:] == [0, 0] and torch.equal(sampled[:1], whole[0][:1])
    untouched = [s for s in range(6) if s != int(x["slots"][0])]
    assert (store.path_len.cpu()[untouched] == -7).all()


def test_streams_and_graphs(dev):
    """A side stream's call equals the default stream's; a captured call replays on new contents of its buffers."""
    from eagle_harness.vllm.tree_accept import sample_tree

    announce("sample tree graph")
    xs = [inputs([8, 5, 8], 8, 2000, BF16, F32, seed=s) for s in (20, 21, 22)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = launch(xs[0], dev)
    side.synchronize()
    check(xs[0], got)
    names = ("logits", "drafted", "cu", "slots", "parents", "coins", "final", "temperature", "q")
    held = {k: xs[0][k].to(dev) for k in names}
    store = Store(6, 8, dev)

    def call():
        return sample_tree(held["logits"], held["drafted"], held["cu"], held["slots"], held["parents"], store, held["coins"],
                           held["final"], held["temperature"], draft_probs=held["q"])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampled, count = call()
    for x in xs + xs:
        for k in names:
            held[k].copy_(x[k])
        store.path.fill_(-7)
        store.path_len.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        check(x, (sampled, count, store))
        launch(x, dev)  # eager work between the replays


@pytest.mark.parametrize("requests,width,vocab,dtype", [(2300, 8, 40, F32), (220, 8, 45000, BF16)])
def test_many_rows(dev, requests, width, vocab, dtype):
    """Batches of more than 2^14 pieces of rows: the trees' first rows are read before the rest."""
    announce(f"sample tree {requests} requests of up to {width} rows, vocab {vocab} {dtype}")
    x = inputs([0 if b % 40 == 7 else 1 + b % 3 if b % 20 == 3 else width for b in range(requests)], width, vocab, dtype, None, seed=9)
    x["temperature"][::9] = 0.0
    x["parents"][x["slots"][5].long(), 2:] = torch.tensor([0, 7, 1, 2, 3, 40][: width - 2], dtype=torch.int32)  # no tree
    chunks = -(-(vocab + 7) // 4096) * int(x["cu"][-1])
    assert chunks >= 1 << 14
    check(x, launch(x, dev))
