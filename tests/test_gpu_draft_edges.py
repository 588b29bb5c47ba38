"""The sampled draft step's operators at the ends of what they take: storage whose offsets pass 32 bits, calls on two streams at a time,
padded requests whose lengths are anything. Every result has to be the ordinary call's, bit for bit."""

import pytest
import torch

import test_gpu_row_attention_fp8 as rows
import test_gpu_sample_rows as sr
from conftest import announce

pytestmark = pytest.mark.gpu

I32 = torch.int32
FAR = 1 << 30  # elements between rows: the third lies 2^31 of them away


def spaced(x, dev, step=FAR):
    """``x`` with its first dimension ``step`` elements apart."""
    store = torch.empty((x.shape[0] - 1) * step + x[0].numel() + 64, dtype=x.dtype, device=dev)
    far = store.as_strided(x.shape, (step, *x.contiguous().stride()[1:]))
    far.copy_(x)
    return far


def rules(dev):
    return (torch.tensor([0.7, 1.0, 1.3], device=dev), torch.tensor([20, 0, 900], dtype=I32, device=dev),
            torch.tensor([0.9, 0.95, 1.0], device=dev), torch.tensor([0.0, 0.0, 1e-4], device=dev))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_logits_far_apart(dev, dtype):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce(f"far rows of logits {dtype}")
    x, coins = sr._logits(3, 5000, dtype, 3).to(dev), torch.rand(3, 4, device=dev)
    probs, cut = torch.empty(3, 5000, device=dev), torch.empty_like(x)
    want = draw_tokens(x, coins, *rules(dev), probs=probs), truncate_logits(x, *rules(dev), out=cut)
    far, out = spaced(x, dev), spaced(torch.zeros_like(probs), dev)
    assert torch.equal(draw_tokens(far, coins, *rules(dev), probs=out), want[0]) and torch.equal(out, probs)
    assert truncate_logits(far, *rules(dev), out=far) is far
    assert torch.equal(far, cut)


@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_far_apart(dev, interleaved):
    from eagle_harness.vllm.rotary import rotary_frequencies, rotate_rows

    announce(f"far heads interleaved={interleaved}")
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randn(3, h, 96, generator=gen).bfloat16().to(dev) for h in (4, 2))
    at, f = torch.tensor([0, 77, 131071], device=dev), rotary_frequencies(64, device=dev)[0]
    far_q, far_k = spaced(q, dev), spaced(k.transpose(0, 1).contiguous(), dev, 2 * FAR).transpose(0, 1)
    rotate_rows(far_q, far_k, at, f, interleaved=interleaved)
    rotate_rows(q, k, at, f, interleaved=interleaved)
    assert torch.equal(far_q, q) and torch.equal(far_k, k)


def test_tables_far_apart(dev):
    from eagle_harness.vllm.page_tables import resize_tables, slot_maps

    announce("far tables")
    ends = []
    for far in (False, True):
        table = torch.arange(30, dtype=I32).view(3, 10)
        table = spaced(table, dev) if far else table.to(dev)
        pages, free = torch.tensor([10, 3, 2], dtype=I32, device=dev), torch.zeros(30, dtype=I32, device=dev)
        num, idx = torch.zeros(1, dtype=I32, device=dev), torch.tensor([2, 0], dtype=I32, device=dev)
        resize_tables(table, pages, idx, torch.tensor([90, 20], device=dev), free, num, 16)
        batch = torch.zeros(2, 10, dtype=I32, device=dev)
        batch = spaced(batch, dev, 2 * FAR + 8) if far else batch
        slots = torch.empty(40, dtype=torch.int64, device=dev)
        slot_maps(table, pages, idx, torch.tensor([60, 0], device=dev), torch.tensor([0, 30, 35], device=dev), 16, slots=slots,
                  batch_table=batch)
        ends.append((table.clone(), pages, free, num, batch.clone(), slots))
    for one, two in zip(*ends):
        assert torch.equal(one, two)
    assert pages.tolist() == [2, 3, 6] and num.tolist() == [4]


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("step,n", [(2, 2), (0, 7)])
def test_pages_far_apart(dev, step, n, dim):
    """Pages past 4 GiB from the cache's start."""
    announce(f"far fp8 pages step={step} dim={dim}")
    gen = torch.Generator().manual_seed(dim + step)
    page, seq = 16, torch.tensor([50, 9], device=dev)
    keys, ks = (t.to(dev) for t in rows._cache(gen, 11, page, 2, dim))
    values, vs = (t.to(dev) for t in rows._cache(gen, 11, page, 2, dim))
    table = torch.randperm(11, generator=gen)[:10].view(2, 5).int().to(dev)
    anc = (table[:, None, 3:4] * page + torch.arange(step, device=dev, dtype=I32)).expand(2, n, step) if step else None
    q = torch.randn(2 * n, 8, dim, generator=gen).bfloat16().to(dev)
    call = dict(rows=n, step=step, window=40, splits=3, table_page=page)
    want = rows._launch(dev, q, keys, values, ks, vs, table, seq, anc, **call)
    wide = (1 << 29) + 1024  # bytes a page: eight of them pass 2^32
    far = [spaced(t.view(torch.uint8), dev, wide).view(torch.float8_e4m3fn) for t in (keys, values)]
    assert torch.equal(rows._launch(dev, q, *far, ks, vs, table, seq, anc, **call), want)


@pytest.mark.parametrize("length", [-(1 << 40), -3, 1 << 31, 1 << 40])
@pytest.mark.parametrize("step", [0, 2])
def test_a_padded_request_of_any_length(dev, step, length):
    """The other request's rows are what they are without it, and the padded one's are numbers."""
    announce(f"fp8 rows: a padded length {length} step={step}")
    gen = torch.Generator().manual_seed(8)
    page, dim, n = 16, 128, 3
    keys, ks = (t.to(dev) for t in rows._cache(gen, 12, page, 2, dim))
    values, vs = (t.to(dev) for t in rows._cache(gen, 12, page, 2, dim))
    table = torch.arange(12, dtype=I32, device=dev).view(2, 6)
    anc = torch.zeros(2, n, step, dtype=I32, device=dev) if step else None
    q = torch.randn(2 * n, 4, dim, generator=gen).bfloat16().to(dev)
    got = [rows._launch(dev, q, keys, values, ks, vs, table, torch.tensor([70, other], device=dev), anc, rows=n, step=step, window=0,
                        splits=2, table_page=page) for other in (11, length)]
    assert torch.equal(got[0][:n], got[1][:n]) and got[1].isfinite().all()


def test_two_streams_at_a_time(dev):
    """Every operator on two streams with inputs of their own, launched in turn without a wait between them."""
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention
    from eagle_harness.vllm.page_tables import resize_tables, slot_maps
    from eagle_harness.vllm.rotary import rotary_frequencies, rotate_rows
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce("two streams")
    f = rotary_frequencies(64, device=dev)[0]
    sides = []
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        keys, ks = (t.to(dev) for t in rows._cache(gen, 80, 16, 2, 128))
        values, vs = (t.to(dev) for t in rows._cache(gen, 80, 16, 2, 128))
        sides.append(dict(
            x=sr._logits(3, 60001, "bf16", seed).to(dev), coins=torch.rand(3, 2, generator=gen).to(dev), q=torch.randn(8, 8, 128, generator=gen).bfloat16().to(dev),
            at=torch.randint(0, 9000, (8,), generator=gen).to(dev), keys=keys, values=values, ks=ks, vs=vs,
            seq=torch.tensor([300 + seed, 90], device=dev), idx=torch.tensor([1, 0], dtype=I32, device=dev), rules=rules(dev)))

    def once(s):
        n = 2 * 8 * 5 * 16
        part, lse = torch.empty(n, 128, device=dev), torch.empty(n, device=dev)
        table, pages = torch.zeros(2, 40, dtype=I32, device=dev), torch.zeros(2, dtype=I32, device=dev)
        free, num = torch.arange(80, dtype=I32, device=dev), torch.full((1,), 80, dtype=I32, device=dev)
        resize_tables(table, pages, s["idx"], s["seq"] + 4, free, num, 16)
        slots, batch = torch.empty(8, dtype=torch.int64, device=dev), torch.empty(2, 40, dtype=I32, device=dev)
        slot_maps(table, pages, s["idx"], s["seq"], s["starts"], 16, slots=slots, batch_table=batch)
        q, out = torch.empty_like(s["q"]), torch.empty_like(s["q"])
        rotate_rows(s["q"], None, s["at"], f, q_out=q)
        rows_attention(q, s["keys"], s["values"], out, part, lse, batch, s["seq"], None, rows_per_request=4, step=0, window=0,
                       scale=128**-0.5, launch=RowsLaunch(splits=4, block_n=32), table_page=16, k_scale=s["ks"], v_scale=s["vs"])
        probs = torch.empty(3, 60001, device=dev)
        tokens = draw_tokens(s["x"], s["coins"], *s["rules"], probs=probs)
        return table, pages, num, slots, batch, q, out, tokens, probs, truncate_logits(s["x"], *s["rules"])

    for s in sides:
        s["starts"] = torch.tensor([0, 4, 8], dtype=I32, device=dev)
    want = [[t.clone() for t in once(s)] for s in sides]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, stream in zip(sides, streams):
            with torch.cuda.stream(stream):
                got.append(once(s))
    torch.cuda.synchronize()
    for i, result in enumerate(got):
        for one, two in zip(result, want[i % 2]):
            assert torch.equal(one, two), i


@pytest.mark.parametrize("p", [0.9, 1.0])
@pytest.mark.parametrize("kind", ["zeros", "few zeros", "large", "small", "masked", "at 64", "wide", "below"])
def test_rows_that_no_rule_bounds(dev, kind, p):
    """Values at the edges of what one pass over a bf16 row can count: many zeros, magnitudes of 64 and more, all of them tiny, masks,
    a hot temperature, all far below 0."""
    announce(f"rows that no rule bounds: {kind} p={p}")
    x, t = sr._logits(3, 20011, "bf16", 17).float(), 1.0
    if kind == "zeros":
        x[:, 100:9000] = 0.0
    elif kind == "few zeros":
        x[:, 100:700] = 0.0
        x[:, 700:900] = -0.0
    elif kind == "large":
        x, t = x * 20, 8.0
    elif kind == "small":
        x = x * 1e-4
    elif kind == "masked":
        x[:, ::3], x[:, 1::9] = -torch.inf, torch.finfo(torch.bfloat16).min
    elif kind == "at 64":
        x[0, 5], x[1, 5], x[2, 5] = 63.75, 64.0, 500.0
    elif kind == "wide":
        t = 3.0
    elif kind == "below":
        x = x - 40.0
    sr._check(dev, x.bfloat16(), t, 0, p, 0.0, probs="f32")
