"""Latent verify attention on the GPU against the 64-bit oracle, element by element within the bound of 16-bit weights and
outputs: head counts and widths of every row split, both ranks, 16-bit and fp8 pages, contexts from none to many splits,
odd pages, masks, values that are not finite, tables out of range, streams and graphs."""

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import latent as olat
from workloads import seeded_tree, tree_masks

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def inputs(contexts, sizes, heads, dtype=BF16, cache="same", rank=512, page=16, seed=0, pow2=True):
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    dim = rank + 64
    starts = torch.tensor([0, *np.cumsum(sizes)], dtype=torch.int32)
    need = [max(1, -(-c // page)) for c in contexts]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.zeros(len(sizes), max(need) + 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    pages = torch.randn(blocks, page, dim, generator=gen)
    scale = None
    if cache == "fp8":
        scale = torch.exp2(torch.randint(-7, 0, (blocks,), generator=gen).float())
        if not pow2:
            scale = scale * (1 + torch.rand(blocks, generator=gen))
        pages = (pages / scale[:, None, None]).clamp(-448, 448).to(FP8)
    else:
        pages = pages.to(dtype)
    width = max(sizes)
    masks = torch.zeros(len(sizes), width, dtype=torch.int64)
    for b, n in enumerate(sizes):
        if n:
            masks[b, :n] = torch.tensor(tree_masks(seeded_tree(rng, n)))
    tokens = int(starts[-1])
    return dict(q=torch.randn(tokens, heads, dim, generator=gen).to(dtype), new=torch.randn(tokens, dim, generator=gen).to(dtype),
                cache=pages, page_scale=scale, table=table, context=torch.tensor(contexts, dtype=torch.int32), starts=starts,
                masks=masks, scale=0.07, rank=rank, width=width)


def launch(x, dev, out=None, **over):
    from eagle_harness.vllm.latent_attention import latent_verify_attention

    y = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in dict(x, **over).items()}
    if out is None:
        out = torch.full((x["q"].shape[0], x["q"].shape[1], x["rank"]), 9.0, dtype=x["q"].dtype, device=dev)
    return latent_verify_attention(y["q"], y["new"], y["cache"], y["table"], y["context"], y["starts"], y["masks"], y["scale"],
                                   out, max_query_len=y["width"], latent_scale=y["page_scale"])


def check(x, got, **over):
    x = dict(x, **over)
    want, bound = olat.latent_attention(x["q"], x["new"], x["cache"], x["table"], x["context"], x["starts"], x["masks"],
                                        x["scale"], x["rank"], x["page_scale"])
    g = got.detach().cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    off = torch.where(torch.isnan(want), 0.0, (g - want).abs() - bound)
    assert float(off.max()) <= 0, f"{float(off.max()):.3g} beyond the bound at {int(off.argmax())}"


@pytest.mark.parametrize("rank", [512, 256])
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (BF16, "fp8"), (F16, "fp8")])
@pytest.mark.parametrize("heads,sizes", [(16, [1, 1, 1]), (8, [1, 2, 1]), (16, [2, 1, 2]), (16, [3, 4, 1]), (5, [7, 16, 2]),
                                         (16, [16, 9, 12]), (128, [1, 1, 1]), (1, [1, 1, 1])])
def test_rows_match_the_oracle(dev, rank, dtype, cache, heads, sizes):
    announce(f"latent rank {rank} {dtype} cache {cache} heads {heads} sizes {sizes}")
    x = inputs([100, 0, 33], sizes, heads, dtype, cache, rank, seed=heads)
    check(x, launch(x, dev))


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("context", [0, 1, 31, 32, 33, 64, 95, 127, 129, 300])
def test_context_lengths(dev, context, cache):
    announce(f"latent context {context} cache {cache}")
    x = inputs([context], [5], 16, BF16, cache, seed=context)
    check(x, launch(x, dev))


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("heads,width", [(16, 1), (16, 2), (16, 4), (16, 16), (128, 1)])
def test_long_contexts_are_cut_and_merged(dev, heads, width, cache):
    announce(f"latent long heads {heads} width {width} cache {cache}")
    x = inputs([5000, 1700], [width, 1], heads, BF16, cache, seed=width)
    check(x, launch(x, dev))


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 100])
def test_page_sizes(dev, page, cache):
    announce(f"latent page {page} cache {cache}")
    x = inputs([1500, 70, 9], [3, 1, 2], 16, BF16, cache, page=page, seed=page)  # page 1: several windows of table entries
    check(x, launch(x, dev))


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("sizes", [[64, 33], [40, 64], [32, 1]])
def test_wide_trees(dev, sizes, cache):
    announce(f"latent sizes {sizes} cache {cache}")
    x = inputs([50, 0], sizes, 8, BF16, cache, seed=sizes[0])
    check(x, launch(x, dev))


def test_scales_of_any_value_and_size(dev):
    announce("latent scales")
    for dtype in (BF16, F16):
        check_x = inputs([200, 77], [4, 2], 16, dtype, "fp8", seed=3, pow2=False)
        check(check_x, launch(check_x, dev))
        two = dict(check_x, page_scale=check_x["page_scale"][:, None].repeat(1, 1))
        assert torch.equal(launch(two, dev), launch(check_x, dev))


def test_many_requests(dev):
    """More requests than one pass of the tile counts, some of them without rows."""
    announce("latent many requests")
    n = 600
    x = inputs([(37 * b) % 90 for b in range(n)], [(b % 3) for b in range(n)], 2, BF16, rank=256, seed=4)
    check(x, launch(x, dev))


def test_more_requests_than_a_launch_takes(dev):
    announce("latent 2100 requests")
    n = 2100
    x = inputs([(5 * b) % 11 for b in range(n)], [1] * n, 1, BF16, rank=256, page=4, seed=4)
    check(x, launch(x, dev))


def test_masks_that_leave_nothing(dev):
    announce("latent empty masks")
    x = inputs([0, 0, 40], [3, 2, 2], 16, BF16, seed=5)
    x["masks"][0, 1] = 0  # sees nothing: zeros
    x["masks"][2, 0] = 0  # sees the context alone
    x["masks"][1, 1] = -1  # bits past the request's rows do not count
    y = dict(x, masks=x["masks"].clone())
    y["masks"][1, 1] = 3
    got = launch(x, dev)
    assert (got[1] == 0).all()
    check(y, got)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(dev, value, cache):
    announce(f"latent value {value} cache {cache}")
    x = inputs([20, 70], [6, 5], 16, BF16, cache, seed=6)
    clean = launch(x, dev)
    x["new"][2, 100] = value  # request 0, row 2
    # what lies behind a context, and in pages of nobody, is not seen
    codes = x["cache"].clone()
    raw = codes.view(torch.uint8) if cache == "fp8" else codes
    block = int(x["table"][0, 1])
    raw[block, 4:] = 127 if cache == "fp8" else value
    used = set(int(v) for b in range(2) for v in x["table"][b, : 2 if b == 0 else 5])
    for p in range(codes.shape[0]):
        if p not in used:
            raw[p] = 127 if cache == "fp8" else value
    got = launch(x, dev, cache=codes)
    sees = [(int(x["masks"][0, r]) >> 2) & 1 == 1 for r in range(6)] + [False] * 5
    assert any(sees) and not all(sees)
    for r, hit in enumerate(sees):
        if hit:
            assert torch.isnan(got[r]).any()
        else:
            assert torch.equal(got[r], clean[r])


def test_pages_outside_the_cache_are_not_seen(dev):
    announce("latent bad pages")
    for cache in ("same", "fp8"):
        x = inputs([100, 40], [3, 2], 16, BF16, cache, seed=7)
        x["table"][0, 2], x["table"][0, 4], x["table"][1, 0] = -1, 1 << 20, x["cache"].shape[0]
        check(x, launch(x, dev))


def test_lengths_past_the_table_are_cut(dev):
    announce("latent context past the table")
    x = inputs([64, 16], [2, 1], 16, BF16, seed=8)
    capacity = x["table"].shape[1] * 16
    x["table"][:, -1] = 0
    got = launch(x, dev, context=torch.tensor([capacity + 500, -3], dtype=torch.int32))
    check(x, got, context=torch.tensor([capacity, 0], dtype=torch.int32))


def test_rows_behind_the_last_request_stay(dev):
    announce("latent rows behind")
    x = inputs([33, 5], [4, 3], 16, BF16, seed=9)
    out = torch.full((7, 16, 512), 3.0, dtype=BF16, device=dev)
    got = launch(x, dev, out, starts=torch.tensor([0, 4, 5], dtype=torch.int32))
    assert (got[5:] == 3).all()
    want = inputs([33, 5], [4, 3], 16, BF16, seed=9)
    cut = dict(want, starts=torch.tensor([0, 4, 5], dtype=torch.int32))
    ref, bound = olat.latent_attention(cut["q"], cut["new"], cut["cache"], cut["table"], cut["context"], cut["starts"],
                                       cut["masks"], cut["scale"], 512)
    assert bool(((got[:5].cpu().double() - ref[:5]).abs() <= bound[:5]).all())
    beyond = launch(x, dev, out.fill_(3.0), starts=torch.tensor([0, 4, 900], dtype=torch.int32))  # rows that are not there
    assert (beyond[4:] == 3).all() and torch.equal(beyond[:4], got[:4])


def test_strided_operands(dev):
    announce("latent strides")
    x = inputs([90, 41], [4, 2], 16, BF16, seed=10)
    q = torch.zeros(6, 16, 640, dtype=BF16, device=dev)[..., :576]
    q.copy_(x["q"])
    new = torch.zeros(6, 3, 576, dtype=BF16, device=dev)[:, 1]
    new.copy_(x["new"])
    blocks = x["cache"].shape[0]
    cache = torch.zeros(blocks, 16, 2, 640, dtype=BF16, device=dev)[:, :, 1, :576]
    cache.copy_(x["cache"])
    masks = torch.zeros(2, 9, dtype=torch.int64, device=dev)[:, :4]
    masks.copy_(x["masks"])
    out = torch.zeros(16, 6, 512, dtype=BF16, device=dev).transpose(0, 1)
    got = launch(x, dev, out, q=q, new=new, cache=cache, masks=masks, starts=x["starts"].long(), context=x["context"].long())
    assert torch.equal(got.contiguous(), launch(x, dev))


def test_large_scores(dev):
    """Scores far apart and far from zero: the running maximum has to move."""
    announce("latent large scores")
    for sign in (1, -1):
        x = inputs([400, 10], [3, 2], 16, BF16, seed=11)
        x["cache"] = (x["cache"].float() * torch.linspace(0.1, 6, 400 // 16 + 2 + 1)[: x["cache"].shape[0], None, None]).to(BF16)
        x["scale"] = sign * 1.5
        check(x, launch(x, dev))


def test_streams_and_graphs(dev):
    from eagle_harness.vllm.latent_attention import latent_verify_attention

    announce("latent graph")
    xs = [inputs([700, 90, 0], [4, 2, 3], 16, BF16, "fp8", seed=s) for s in (40, 41, 42)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = launch(xs[0], dev)
    side.synchronize()
    check(xs[0], got)
    names = ("q", "new", "cache", "table", "context", "starts", "masks", "page_scale")
    held = {k: xs[0][k].to(dev) for k in names}
    out = torch.empty(9, 16, 512, dtype=BF16, device=dev)

    def call():
        latent_verify_attention(held["q"], held["new"], held["cache"], held["table"], held["context"], held["starts"],
                                held["masks"], 0.07, out, max_query_len=4, latent_scale=held["page_scale"])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for x in xs + xs:
        for k in names:
            held[k].copy_(x[k])
        graph.replay()
        torch.cuda.synchronize()
        eager = launch(x, dev)
        assert torch.equal(out, eager)
        check(x, out)


def test_two_calls_at_once(dev):
    """Each call has its own workspace: calls on two streams do not disturb each other."""
    announce("latent two streams")
    xs = [inputs([3000], [4], 16, BF16, seed=s) for s in (50, 51)]
    want = [launch(x, dev) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(launch(xs[i], dev))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
