"""fp8 page writes and reads on the GPU against the oracle, byte for byte: page sizes that end inside rows, scales that grow,
accepted paths, infinities and NaN, tables and pages out of range, packed and strided layouts."""

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import kv_pages as okv

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def batch(contexts, counts, heads, dim, page, dtype, seed, spare=3):
    gen = torch.Generator().manual_seed(seed)
    starts = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32)
    need = [max(1, -(-(c + n) // page)) for c, n in zip(contexts, counts)]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(counts), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    cache = torch.randint(0, 256, (blocks, page, heads, dim), generator=gen, dtype=torch.uint8)
    cache = torch.where((cache & 127) == 127, torch.zeros_like(cache), cache).view(FP8)
    scale = torch.exp2(torch.randint(-9, 2, (blocks, heads), generator=gen).float())
    key = torch.randn(int(starts[-1]), heads, dim, generator=gen) * torch.exp2(
        torch.randint(-6, 7, (int(starts[-1]), heads, 1), generator=gen).float())
    return dict(key=key.to(dtype), cache=cache, scale=scale, table=table, context=torch.tensor(contexts, dtype=torch.int32),
                starts=starts, most=max(counts), blocks=blocks)


def same(got, want):
    """Equal bytes; NaN codes of either sign are one."""
    g, w = got.cpu().view(torch.uint8), want.cpu().view(torch.uint8)
    return bool(((g == w) | (((g & 127) == 127) & ((w & 127) == 127))).all())


def write(x, dev, key=None, cache=None, scale=None, value=None, **more):
    from eagle_harness.vllm.kv_pages import write_kv_pages

    key = x["key"].to(dev) if key is None else key
    cache = x["cache"].to(dev) if cache is None else cache
    scale = x["scale"].to(dev) if scale is None else scale
    write_kv_pages(key, None, cache, None, scale, None, x["table"].to(dev), x["context"].to(dev), x["starts"].to(dev),
                   max_query_len=x["most"], **more)
    return cache, scale


def check(x, got, **more):
    cache, scale = x["cache"].clone(), x["scale"].clone()
    okv.write_pages(x["key"], cache, scale, x["table"], x["context"], x["starts"], **more)
    assert torch.equal(got[1].cpu(), scale), "scales"
    assert same(got[0], cache), "codes"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,dim,page", [(4, 256, 16), (1, 576, 64), (2, 64, 24), (8, 128, 16), (1, 40, 1), (3, 7, 5),
                                            (2, 264, 40)])
def test_rows_match_the_oracle(dev, dtype, heads, dim, page):
    announce(f"write pages heads {heads} dim {dim} page {page} {dtype}")
    x = batch([0, 5, page, 3 * page - 1, 17], [1, 2 * page + 3, 0, 2, 3 * page], heads, dim, page, dtype, seed=dim)
    check(x, write(x, dev))


def test_values_and_packed_caches(dev):
    """K and V adjacent in one [blocks, heads, page, 2 D] cache, rows the views of a fused projection's output."""
    from eagle_harness.vllm.kv_pages import write_kv_pages
    from eagle_harness.vllm.tree_attention import split_kv_cache

    announce("write pages packed")
    heads, dim, page = 4, 128, 16
    x = batch([9, 40], [13, 4], heads, dim, page, BF16, seed=1)
    y = batch([9, 40], [13, 4], heads, dim, page, BF16, seed=2)
    both = torch.zeros(x["blocks"], heads, page, 2 * dim, dtype=torch.uint8, device=dev).view(FP8)
    key_cache, value_cache = split_kv_cache(both, dim)
    key_cache.copy_(x["cache"].to(dev))
    value_cache.copy_(y["cache"].to(dev))
    fused = torch.cat([x["key"], torch.zeros_like(x["key"]), y["key"]], 1).to(dev)
    scales = torch.stack([x["scale"], y["scale"]], -1).to(dev)  # [blocks, heads, 2]
    write_kv_pages(fused[:, :heads], fused[:, 2 * heads :], key_cache, value_cache, scales[..., 0], scales[..., 1],
                   x["table"].to(dev), x["context"].to(dev), x["starts"].to(dev), max_query_len=13)
    check(x, (key_cache.contiguous(), scales[..., 0]))
    y["table"] = x["table"]
    check(y, (value_cache.contiguous(), scales[..., 1]))


@pytest.mark.parametrize("offset", [1, 4])
def test_unaligned_rows(dev, offset):
    announce(f"write pages offset {offset}")
    x = batch([3], [20], 2, 64, 16, BF16, seed=7)
    held = torch.zeros(20 * 2 * 64 + 16, dtype=BF16, device=dev)
    key = held[offset : offset + 20 * 128].view(20, 2, 64)
    key.copy_(x["key"])
    check(x, write(x, dev, key=key))


def test_accepted_paths(dev):
    announce("write pages path")
    x = batch([30, 0, 15, 64], [8, 8, 8, 8], 2, 128, 16, BF16, seed=4)
    path = torch.tensor([[0, 1, 2, 3, 4, 5, 6, 7], [0, 2, 5, 7, -1, 0, 0, 0], [0, 0, 0, 0, 0, 0, 0, 0], [0, 3, 9, -4, 6, 0, 0, 0],
                         [0, 1, 4, 0, 0, 0, 0, 0]], dtype=torch.int32)
    path_len = torch.tensor([8, 4, 0, 5, 3], dtype=torch.int32)
    slots = torch.tensor([1, 0, 2, 3], dtype=torch.int64)
    got = write(x, dev, idx_mapping=slots.to(dev), path=path.to(dev), path_len=path_len.to(dev))
    check(x, got, path=path, path_len=path_len, slots=slots)


def test_slots_outside_the_path_table_write_nothing(dev):
    announce("write pages slots out of range")
    x = batch([30, 4], [4, 4], 1, 64, 16, BF16, seed=4)
    path = torch.zeros(2, 4, dtype=torch.int32)
    got = write(x, dev, idx_mapping=torch.tensor([-1, 7]).to(dev), path=path.to(dev),
                path_len=torch.tensor([4, 4], dtype=torch.int32).to(dev))
    assert torch.equal(got[1].cpu(), x["scale"]) and same(got[0], x["cache"])


def test_growth_moves_earlier_rows_without_rounding(dev):
    """One row at a time, each larger than the last: the page's rows end where one write of them all would have put them,
    but for values below the normal range of the last scale."""
    announce("write pages growth")
    n, page, dim = 16, 16, 64
    gen = torch.Generator().manual_seed(9)
    rows = (torch.rand(n, 1, dim, generator=gen) + 0.5) * torch.exp2(torch.arange(n).float() / 3)[:, None, None]
    x = batch([0], [n], 1, dim, page, F32, seed=3)
    x["key"] = rows
    whole = write(x, dev)
    cache, scale = x["cache"].to(dev), x["scale"].to(dev)
    for j in range(n):
        y = dict(x, key=rows[j : j + 1], context=torch.tensor([j], dtype=torch.int32), starts=torch.tensor([0, 1]), most=1)
        write(y, dev, cache=cache, scale=scale)
    assert torch.equal(scale, whole[1])
    block = int(x["table"][0, 0])
    a, b = cache[block].float().cpu(), whole[0][block].float().cpu()
    normal = b.abs() >= 2.0 ** -6
    assert normal.float().mean() > 0.9 and torch.equal(a[normal], b[normal])


def test_infinities_nan_zeros_and_extremes(dev):
    announce("write pages special values")
    x = batch([3, 0, 0, 0, 16], [6, 16, 5, 5, 2], 2, 64, 16, F32, seed=5)
    inf, nan = float("inf"), float("nan")
    x["key"][1, 0, 3], x["key"][2, 1, 4], x["key"][4, 0, 7] = inf, -inf, nan
    x["key"][6:22] = 0.0                       # a page of zeros: scale 0
    x["key"][22:27] *= 1e-40                   # subnormals
    x["key"][27:32] = x["key"][27:32].sign() * 3e38
    x["key"][32, 0, :] = 448.0                 # the largest code exactly
    x["key"][33, 1, :] = 448.0 * (1 + 2.0 ** -23)  # just above: the next scale
    check(x, write(x, dev))


def test_tables_and_pages_out_of_range(dev):
    announce("write pages bad pages")
    x = batch([0, 20, 40], [40, 40, 40], 1, 64, 16, BF16, seed=6)
    x["table"][0, 1] = x["blocks"]
    x["table"][1, 2] = -9
    x["table"][2, 0] = 1 << 30  # a page of the context: not touched
    x["table"] = x["table"][:, :4]  # too short for the last request's rows
    check(x, write(x, dev))
    negative = dict(x, context=torch.tensor([-5, -1, -40], dtype=torch.int32))
    got = write(negative, dev)
    assert torch.equal(got[1].cpu(), x["scale"]) and same(got[0], x["cache"])


def test_more_rows_than_announced_stay_out(dev):
    announce("write pages max rows")
    x = batch([4], [40], 1, 64, 16, BF16, seed=6)
    x["most"] = 21
    check(x, write(x, dev), max_rows=21)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,dim,page", [(4, 256, 16), (1, 576, 64), (2, 64, 24), (3, 7, 5), (1, 40, 1)])
def test_reads_match_the_oracle(dev, dtype, heads, dim, page):
    from eagle_harness.vllm.kv_pages import read_kv_pages

    announce(f"read pages heads {heads} dim {dim} page {page} {dtype}")
    lens = [1, 0, 2 * page + 1, 100, page]
    x = batch(lens, [0] * 5, heads, dim, page, dtype, seed=dim)
    x["table"][3, 2] = x["blocks"] + 5  # a page that is not there reads as zeros
    starts = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32)
    out = torch.full((int(starts[-1]) + 3, heads, dim), 5.0, dtype=dtype, device=dev)
    value = torch.full_like(out, 6.0)
    read_kv_pages(x["cache"].to(dev), x["cache"].flip(0).to(dev), x["scale"].to(dev), x["scale"].flip(0).contiguous().to(dev),
                  x["table"].to(dev), starts.to(dev), out, value, max_len=max(lens))
    for got, cache, scale, rest in ((out, x["cache"], x["scale"], 5.0), (value, x["cache"].flip(0), x["scale"].flip(0), 6.0)):
        want = okv.read_pages(cache, scale, x["table"], starts)
        assert torch.equal(got[:-3].cpu(), want.to(dtype))  # a code times a power of two: one rounding at most
        assert (got[-3:] == rest).all()


def test_expanded_scales_read(dev):
    """A per-tensor scale as a stride-0 view, any fp32 value: one rounded product."""
    from eagle_harness.vllm.kv_pages import read_kv_pages

    announce("read pages expanded scales")
    x = batch([50], [0], 2, 128, 16, F32, seed=2)
    scale = torch.full((1, 1), 0.0173, device=dev).expand(x["blocks"], 2)
    out = torch.empty(50, 2, 128, device=dev)
    read_kv_pages(x["cache"].to(dev), None, scale, None, x["table"].to(dev), torch.tensor([0, 50], device=dev), out, None,
                  max_len=50)
    want = okv.read_pages(x["cache"], scale.cpu(), x["table"], torch.tensor([0, 50]))
    assert torch.equal(out.cpu(), want.float())


def test_streams_and_graphs(dev):
    announce("write pages graph")
    x = batch([9, 33, 2], [7, 3, 5], 4, 128, 16, BF16, seed=11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = write(x, dev)
    side.synchronize()
    check(x, got)
    from eagle_harness.vllm.kv_pages import write_kv_pages

    key, cache, scale = x["key"].to(dev), x["cache"].to(dev), x["scale"].to(dev)
    table, context, starts = x["table"].to(dev), x["context"].to(dev), x["starts"].to(dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        write_kv_pages(key, None, cache, None, scale, None, table, context, starts, max_query_len=7)
    for s in range(4):
        y = batch([9, 33, 2], [7, 3, 5], 4, 128, 16, BF16, seed=30 + s)
        y.update(table=x["table"])
        key.copy_(y["key"])
        cache.copy_(y["cache"])
        scale.copy_(y["scale"])
        graph.replay()
        torch.cuda.synchronize()
        check(y, (cache, scale))
        write(x, dev)
