"""Latent verify attention at the ends of its caches and schedules."""

import pytest
import torch

import test_gpu_latent_attention as lat
from conftest import announce
from oracle import latent as olat

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("heads", [16, 40])
def test_a_cache_of_no_pages(dev, cache, heads):
    """Every page id lies outside it: the round's rows alone are seen, behind a context of many tiles."""
    announce(f"latent cache of no pages {cache} heads {heads}")
    x = lat.inputs([700, 40], [4, 2], heads, BF16, cache, seed=71)
    x["cache"] = x["cache"][:0]
    x["page_scale"] = None if cache == "same" else x["page_scale"][:1]  # (none at all: no pointer, refused)
    x["table"][0, 7], x["table"][0, 9] = -3, 1 << 30
    lat.check(x, lat.launch(x, dev))


def crowded(x):
    """``x`` with one more request behind it, of one row and a long context over one page: enough tiles that workgroups take 64
    query rows (where a request has more than 32), on the short contexts in front."""
    page = x["cache"].shape[1]
    keys = 32 * 650
    table = torch.cat([x["table"], torch.zeros(x["table"].shape[0], -(-keys // page), dtype=torch.int32)], 1)
    row = torch.full((1, table.shape[1]), int(x["table"][0, 0]), dtype=torch.int32)
    mask = torch.zeros(1, x["masks"].shape[1], dtype=torch.int64)
    mask[0, 0] = 1
    return dict(x, q=torch.cat([x["q"], x["q"][-1:]]), new=torch.cat([x["new"], x["new"][-1:]]), table=torch.cat([table, row]),
                context=torch.cat([x["context"], torch.tensor([keys], dtype=torch.int32)]),
                starts=torch.cat([x["starts"], x["starts"][-1:] + 1]), masks=torch.cat([x["masks"], mask]))


def check_both(x, dev, **over):
    """On its own (16 rows a workgroup, or what the widest request fills) and in a crowd."""
    lat.check(x, lat.launch(x, dev, **over))
    lat.check(x, lat.launch(crowded(x), dev, **over)[:-1])


@pytest.mark.parametrize("rank", [512, 256])
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (BF16, "fp8"), (F16, "fp8")])
@pytest.mark.parametrize("heads,sizes", [(16, [3, 4, 1]), (5, [7, 16, 2]), (16, [16, 9, 12]), (128, [1, 1, 1]), (8, [64, 33, 0])])
def test_forms_of_rows(dev, rank, dtype, cache, heads, sizes):
    announce(f"latent forms rank {rank} {dtype} cache {cache} heads {heads} sizes {sizes}")
    check_both(lat.inputs([100, 0, 33], sizes, heads, dtype, cache, rank, seed=heads), dev)


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("context", [0, 1, 31, 32, 33, 64, 95, 127, 129, 300])
def test_forms_of_contexts(dev, context, cache):
    announce(f"latent forms context {context} cache {cache}")
    check_both(lat.inputs([context], [5], 16, BF16, cache, seed=context), dev)


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("page", [1, 3, 24, 100])
def test_forms_of_pages(dev, page, cache):
    announce(f"latent forms page {page} cache {cache}")
    check_both(lat.inputs([1500, 70, 9], [3, 1, 2], 16, BF16, cache, page=page, seed=page), dev)


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("rank", [512, 256])
def test_forms_of_two_tiles_of_rows(dev, cache, rank):
    announce(f"latent forms two tiles of rows cache {cache} rank {rank}")
    check_both(lat.inputs([0, 32, 64, 96, 128, 160, 192, 224, 250], [64, 33, 64, 40, 64, 64, 50, 64, 37], 4, BF16, cache,
                          rank=rank, seed=73), dev)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_forms_of_scales(dev, dtype):
    announce(f"latent forms scales {dtype}")
    check_both(lat.inputs([200, 77], [4, 2], 16, dtype, "fp8", seed=74, pow2=False), dev)


@pytest.mark.parametrize("sign", [1, -1])
def test_forms_of_large_scores(dev, sign):
    announce(f"latent forms large scores {sign}")
    x = lat.inputs([400, 10], [3, 2], 16, BF16, seed=75)
    x["cache"] = (x["cache"].float() * torch.linspace(0.1, 6, x["cache"].shape[0])[:, None, None]).to(BF16)
    x["scale"] = sign * 1.5
    check_both(x, dev)


def test_forms_of_masks_and_bad_pages(dev):
    announce("latent forms masks and bad pages")
    x = lat.inputs([0, 100, 40], [3, 4, 2], 16, BF16, seed=76)
    x["masks"][0, 1] = 0  # sees nothing: zeros
    x["masks"][2, 0] = 0  # sees the context alone
    x["table"][1, 2], x["table"][1, 4], x["table"][2, 0] = -1, 1 << 20, x["cache"].shape[0]
    check_both(x, dev)
    assert (lat.launch(crowded(x), dev)[1] == 0).all()


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_forms_of_values_that_are_not_finite(dev, value, cache):
    announce(f"latent forms value {value} cache {cache}")
    x = lat.inputs([20, 70], [6, 5], 16, BF16, cache, seed=77)
    for form in (lambda y: y, crowded):
        clean = lat.launch(form(x), dev)
        y = dict(x, new=x["new"].clone())
        y["new"][2, 100] = value  # request 0, row 2
        got = lat.launch(form(y), dev)
        sees = [(int(x["masks"][0, r]) >> 2) & 1 == 1 for r in range(6)] + [False] * 5
        assert any(sees) and not all(sees)
        for r, hit in enumerate(sees):
            assert torch.isnan(got[r]).any() if hit else torch.equal(got[r], clean[r])


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("heads,sizes,contexts", [(128, [1], [2000]), (16, [16], [900]), (16, [4, 2, 4], [500, 0, 130]),
                                                  (16, [1, 1], [3000, 40]), (16, [2, 1], [700, 90]), (32, [8] * 8, [2600] * 8)])
def test_the_tables_width_changes_nothing(dev, heads, sizes, contexts, cache):
    """The contexts decide how rows and tiles are shared out, not the blocks that a table has room for."""
    announce(f"latent wide tables heads {heads} sizes {sizes} cache {cache}")
    x = lat.inputs(contexts, sizes, heads, BF16, cache, seed=78)
    want = lat.launch(x, dev)
    for more in (300, 2048, 8192):
        wide = torch.cat([x["table"], torch.zeros(len(sizes), more, dtype=torch.int32)], 1)
        assert torch.equal(lat.launch(dict(x, table=wide), dev), want)


def test_a_captured_call_takes_each_batch_in_its_own_form(dev):
    """One graph replayed on short and on long contexts: the choice is made on the GPU."""
    from eagle_harness.vllm.latent_attention import latent_verify_attention

    announce("latent forms graph")
    xs = [lat.inputs(c, [4, 3], 16, BF16, "fp8", seed=s) for s, c in ((79, [60, 9]), (80, [21000, 700]), (81, [0, 300]))]
    blocks, columns = max(x["cache"].shape[0] for x in xs), max(x["table"].shape[1] for x in xs)
    for x in xs:
        more = blocks - x["cache"].shape[0]
        x["cache"] = torch.cat([x["cache"], x["cache"][:1].expand(more, -1, -1)])
        x["page_scale"] = torch.cat([x["page_scale"], torch.ones(more)])
        x["table"] = torch.cat([x["table"], torch.zeros(2, columns - x["table"].shape[1], dtype=torch.int32)], 1)
    names = ("q", "new", "cache", "table", "context", "starts", "masks", "page_scale")
    held = {k: xs[0][k].to(dev) for k in names}
    out = torch.empty(7, 16, 512, dtype=BF16, device=dev)

    def call():
        latent_verify_attention(held["q"], held["new"], held["cache"], held["table"], held["context"], held["starts"],
                                held["masks"], 0.07, out, max_query_len=4, latent_scale=held["page_scale"])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    want = [lat.launch(x, dev) for x in xs]
    for i in (0, 1, 2, 1, 0):
        for k in names:
            held[k].copy_(xs[i][k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    lat.check(xs[0], want[0])
    lat.check(xs[2], want[2])


@pytest.mark.parametrize("power", [7, 8, 9, 12, 14])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scales_of_large_values(dev, dtype, power):
    """A page scaled for values near fp16's largest, and beyond, in a column that no query looks at."""
    announce(f"latent large scales 2^{power} {dtype}")
    x = lat.inputs([320, 50], [4, 2], 16, dtype, "fp8", seed=82)
    x["q"][..., 5] = 0
    block = int(x["table"][0, 3])
    codes = torch.zeros(16, 576)
    codes[:, ::7] = 2.0 ** -9  # the smallest code
    codes[2, 5] = 256.0 if power == 8 else 448.0
    x["cache"][block] = codes.to(x["cache"].dtype)
    x["page_scale"][block] = 2.0 ** power
    want, bound = olat.latent_attention(x["q"], x["new"], x["cache"], x["table"], x["context"], x["starts"], x["masks"],
                                        x["scale"], x["rank"], x["page_scale"])
    # Outputs beyond the type: fp16 ends at 65504, its step there is 32, and from 65520, half a step on, a value rounds to infinity.
    beyond = (want.abs() + bound >= 65520) & (dtype == F16)
    for got in (lat.launch(x, dev), lat.launch(crowded(x), dev)[:-1]):
        g = got.cpu().double()
        g = torch.where(beyond & torch.isinf(g) & (g * want > 0), want, g)
        assert float(((g - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype,powers", [(F16, (-14, -20, -26, -33)), (BF16, (-60, -100, -110, -118))])
def test_scales_of_small_values(dev, dtype, powers):
    """Values below fp16's subnormals still make scores: queries and scale as large as the values are small."""
    for power in powers:
        announce(f"latent small scales 2^{power} {dtype}")
        x = lat.inputs([320, 50], [4, 2], 16, dtype, "fp8", seed=83)
        x["page_scale"][:] = 2.0 ** power
        x["cache"] = (torch.randn(x["cache"].shape, generator=torch.Generator().manual_seed(83)) * 20).to(x["cache"].dtype)
        x["new"] = x["new"] * 0
        x["scale"] = 0.002 * 2.0 ** -power
        small_check(x, dev)


def small_check(x, dev):
    """Within the oracle's bound and, in fp16, what its subnormals allow: an output below 2^-14 is rounded to a multiple of 2^-24,
    off by 2^-25 at most; and a weight p times the part r of its scale below 2^-15 is, so o is off by at most 2^-25 / r a key, of
    the values' r |c| = 2^-15 |code|, over a sum of weights of at least 1/2."""
    want, bound = olat.latent_attention(x["q"], x["new"], x["cache"], x["table"], x["context"], x["starts"], x["masks"],
                                        x["scale"], x["rank"], x["page_scale"])
    if x["q"].dtype == F16:
        keys = int(x["context"].max()) + x["width"]
        bound = bound + 2.0 ** -25 + 2 * keys * 2.0 ** -25 * 2.0 ** -15 * float(x["cache"].float().abs().max())
    for got in (lat.launch(x, dev), lat.launch(crowded(x), dev)[:-1]):
        assert float(((got.cpu().double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype,powers", [(F16, (-14, -20, -26, -33)), (BF16, (-60, -100, -110, -118))])
def test_keys_of_small_values_beside_ordinary_ones(dev, dtype, powers):
    """Queries look at one half of the columns, the round's rows have values in the other: what the small keys' scores take from
    the rows' weights shows in ordinary numbers."""
    for power in powers:
        announce(f"latent small scales 2^{power} beside ordinary rows {dtype}")
        x = lat.inputs([320, 50], [4, 2], 16, dtype, "fp8", seed=84)
        x["page_scale"][:] = 2.0 ** power
        x["cache"] = (torch.randn(x["cache"].shape, generator=torch.Generator().manual_seed(84)) * 20).to(x["cache"].dtype)
        x["q"][..., :288] = 0
        x["new"][:, 288:] = 0
        x["scale"] = 0.006 * 2.0 ** -power
        small_check(x, dev)


def test_launches_of_many_requests_choose_for_themselves(dev):
    """More requests than one launch takes, the first launch with much to do and the last with little."""
    announce("latent forms over several launches")
    n = 1100
    x = lat.inputs([(37 * b) % 60 for b in range(n)], [b % 3 for b in range(n)], 24, BF16, rank=256, seed=85)
    lat.check(x, lat.launch(x, dev))
