"""Calls of the sampled, quantized round's operators beside the ordinary ones: vocabularies of many pieces, walks that are rejected
again and again, calls on two streams at once, large batches replayed, rows wider than a workgroup, empty batches, tables of
either width, trees of two tiles behind contexts of any number of tiles."""

import numpy as np
import pytest
import torch

import test_gpu_kv_pages as kv
import test_gpu_latent_attention as lat
import test_gpu_sample_tree as st
from conftest import announce
from oracle import kv_pages as okv

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype,probs", [(BF16, None), (F32, None), (BF16, F32)])
def test_large_vocabularies(dev, dtype, probs):
    announce(f"sample tree vocab 300001 {dtype} probs {probs}")
    x = st.inputs([4, 3, 2], 4, 300001, dtype, probs, seed=31)
    x["final"] = torch.tensor([0.999, 0.5, 0.0])
    x["temperature"][1] = 8.0  # flat: the token lies anywhere
    st.check(x, st.launch(x, dev))


@pytest.mark.parametrize("dtype,probs,vocab", [(BF16, F32, 20000), (F32, F32, 5000), (BF16, None, 20000)])
def test_walks_rejected_again_and_again(dev, dtype, probs, vocab):
    announce(f"sample tree rejections vocab {vocab} {dtype} probs {probs}")
    x = st.inputs([12, 16, 9, 16], 16, vocab, dtype, probs, seed=32)
    for b in range(4):  # all of the root's children but the last lose; a tree below it
        slot, n = int(x["slots"][b]), int(x["cu"][b + 1] - x["cu"][b])
        x["parents"][slot, 1:n] = torch.tensor([0] * 6 + [r - 3 for r in range(7, n)], dtype=torch.int32)[: n - 1]
        x["coins"][int(x["cu"][b]) + 1 : int(x["cu"][b]) + 6] = 0.9999
        x["coins"][int(x["cu"][b]) + 6] = 0.0
    st.check(x, st.launch(x, dev))


@pytest.mark.parametrize("probs", [None, F32])
def test_sampled_walks_at_once(dev, probs):
    announce(f"sample tree two streams probs {probs}")
    xs = [st.inputs([16, 7], 16, 30000, BF16, probs, seed=s) for s in (33, 34)]
    for x in xs:
        st.check(x, st.launch(x, dev))
    on = [{k: v.to(dev) for k, v in x.items() if isinstance(v, torch.Tensor)} for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(st.launch(dict(xs[i], **on[i]), dev))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            st.check(xs[i], g)


def test_a_large_batch_replays(dev):
    from eagle_harness.vllm.tree_accept import sample_tree

    announce("sample tree large batch captured")
    xs = [st.inputs([8] * 2300, 8, 40, F32, None, seed=s) for s in (35, 36)]
    names = ("logits", "drafted", "cu", "slots", "parents", "coins", "final", "temperature")
    held = {k: xs[0][k].to(dev) for k in names}
    store = st.Store(2303, 8, dev)

    def call():
        return sample_tree(held["logits"], held["drafted"], held["cu"], held["slots"], held["parents"], store, held["coins"],
                           held["final"], held["temperature"])

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
        st.check(x, (sampled, count, store))


@pytest.mark.parametrize("heads,dim", [(20, 128), (33, 64), (9, 264), (300, 3)])
def test_rows_wider_than_a_workgroup(dev, heads, dim):
    from eagle_harness.vllm.kv_pages import read_kv_pages

    announce(f"pages of {heads} heads x {dim}")
    x = kv.batch([5, 0, 30], [9, 20, 3], heads, dim, 16, BF16, seed=heads)
    got = kv.write(x, dev)
    kv.check(x, got)
    lens = [14, 20, 33]
    starts = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32)
    out = torch.empty(sum(lens), heads, dim, dtype=BF16, device=dev)
    read_kv_pages(got[0], None, got[1], None, x["table"].to(dev), starts.to(dev), out, None, max_len=40)
    assert torch.equal(out.cpu(), okv.read_pages(got[0].cpu(), got[1].cpu(), x["table"], starts).to(BF16))


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("rank", [512, 256])
def test_trees_of_two_tiles_behind_any_context(dev, cache, rank):
    announce(f"latent two tiles of rows, cache {cache} rank {rank}")
    x = lat.inputs([0, 32, 64, 96, 128, 160, 192, 224, 250], [64, 33, 64, 40, 64, 64, 50, 64, 37], 4, BF16, cache, rank=rank,
                   seed=37)
    lat.check(x, lat.launch(x, dev))


def test_tables_of_either_width(dev):
    announce("latent int64 tables")
    x = lat.inputs([90, 3], [4, 2], 16, BF16, seed=38)
    y = dict(x, context=x["context"].long(), starts=x["starts"].long())
    assert torch.equal(lat.launch(y, dev), lat.launch(x, dev))


def test_empty_batches(dev):
    announce("empty batches")
    x = lat.inputs([90, 3], [1, 2], 16, BF16, seed=39)
    none = dict(x, q=x["q"][:0], new=x["new"][:0], starts=torch.zeros(3, dtype=torch.int32))
    assert lat.launch(none, dev).shape[0] == 0
    no_requests = dict(x, starts=torch.zeros(1, dtype=torch.int32))
    assert (lat.launch(no_requests, dev) == 9.0).all()
    y = st.inputs([3, 2], 4, 50, F32, None, seed=40)
    y["cu"] = torch.zeros(1, dtype=torch.int32)
    sampled, count, store = st.launch(y, dev)
    assert sampled.shape == (0, 4) and count.shape == (0,) and (store.path_len == -7).all()
    z = kv.batch([5, 40], [2, 3], 4, 128, 16, BF16, seed=41)
    z["starts"] = torch.zeros(3, dtype=torch.int32)
    kv.check(z, kv.write(z, dev))
    z["starts"] = torch.zeros(1, dtype=torch.int32)
    got = kv.write(z, dev)
    assert kv.same(got[0], z["cache"]) and torch.equal(got[1].cpu(), z["scale"])


def test_batches_of_no_rows(dev):
    """Requests, but no row among them: the walks are empty, pages and scales stay."""
    announce("batches of no rows")
    y = st.inputs([0, 0], 4, 50, F32, F32, seed=42)
    st.check(y, st.launch(y, dev))
    z = kv.batch([5, 40], [0, 0], 4, 128, 16, BF16, seed=43)
    got = kv.write(z, dev)
    assert kv.same(got[0], z["cache"]) and torch.equal(got[1].cpu(), z["scale"])
    from eagle_harness.vllm.kv_pages import read_kv_pages

    out = torch.empty(0, 4, 128, dtype=BF16, device=dev)
    read_kv_pages(z["cache"].to(dev), None, z["scale"].to(dev), None, z["table"].to(dev), z["starts"].to(dev), out, None,
                  max_len=8)


@pytest.fixture
def wide_tables(monkeypatch):
    """Inputs whose tables could hold contexts far longer than they do: what the tables allow decides how many query rows a
    workgroup takes, so these run the forms of long contexts on the short ones of the tests."""
    plain = lat.inputs

    def padded(*args, page=16, **kw):
        x = plain(*args, page=page, **kw)
        more = torch.zeros(x["table"].shape[0], -(-1100 * 32 // page), dtype=torch.int32)
        return dict(x, table=torch.cat([x["table"], more], 1))

    monkeypatch.setattr(lat, "inputs", padded)


@pytest.mark.parametrize("rank", [512, 256])
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (BF16, "fp8"), (F16, "fp8")])
@pytest.mark.parametrize("heads,sizes", [(16, [3, 4, 1]), (5, [7, 16, 2]), (16, [16, 9, 12]), (128, [1, 1, 1])])
def test_long_tables(dev, wide_tables, rank, dtype, cache, heads, sizes):
    lat.test_rows_match_the_oracle(dev, rank, dtype, cache, heads, sizes)


@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_long_tables_of_any_context(dev, wide_tables, cache):
    for context in (0, 1, 31, 32, 33, 64, 95, 127, 129, 300):
        lat.test_context_lengths(dev, context, cache)
    for page in (1, 3, 24, 100):
        lat.test_page_sizes(dev, page, cache)
    for sizes in ([64, 33], [40, 64], [32, 1]):
        lat.test_wide_trees(dev, sizes, cache)
    test_trees_of_two_tiles_behind_any_context(dev, cache, 512)
    for value in (float("nan"), float("inf")):
        lat.test_values_that_are_not_finite_reach_only_rows_that_see_them(dev, value, cache)


def test_long_tables_of_every_other_kind(dev, wide_tables):
    lat.test_scales_of_any_value_and_size(dev)
    lat.test_masks_that_leave_nothing(dev)
    lat.test_pages_outside_the_cache_are_not_seen(dev)
    lat.test_rows_behind_the_last_request_stay(dev)
    lat.test_strided_operands(dev)
    lat.test_large_scores(dev)
    lat.test_streams_and_graphs(dev)
