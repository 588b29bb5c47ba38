"""Drawn tokens, their distributions and truncated rows on the GPU against the oracle in 64 bits.

Tokens and kept parts are decisions and have to be equal. Probabilities: a weight computed in 64 bits over a sum of masses that
are off by 2^-46 of the largest each, so the rounding to the output's type is all that counts: 2^-24 (fp32), 2^-11 (fp16,
or half its smallest step, 2^-25), 2^-8 / 2 (bf16) of the value; a hundredth of that is added for the sum."""

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import sampling as ora

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}


def _logits(rows, vocab, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=gen) * spread
    for r in range(rows):
        at = torch.randint(0, vocab, (min(vocab, 12),), generator=gen)
        x[r, at] = 6.0 + 2.0 * torch.randn(len(at), generator=gen)
    return x.to(DTYPES[dtype])


def _rules(rows, t, k, p, m, dev):
    full = lambda v, d: torch.full((rows,), v, dtype=d, device=dev)  # noqa: E731
    return full(t, torch.float32), full(k, torch.int32), full(p, torch.float32), full(m, torch.float32)


def _check(dev, logits, t, k, p, m, *, coins=None, probs=None, entries=None, place=None):
    """Draws, probabilities and the truncated rows of ``logits`` (on the CPU) under rules given as numbers or vectors."""
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    rows, vocab = logits.shape
    here = logits.to(dev) if place is None else place(logits)
    vec = lambda v, d: torch.as_tensor(v, dtype=d).expand(rows).contiguous() if not torch.is_tensor(v) else v  # noqa: E731
    t, k, p, m = vec(t, torch.float32), vec(k, torch.int32), vec(p, torch.float32), vec(m, torch.float32)
    on = [v.to(dev) for v in (t, k, p, m)]
    if coins is None:
        coins = torch.rand(rows, 3, generator=torch.Generator().manual_seed(vocab))
    of = torch.arange(rows) if entries is None else entries
    out = None if probs is None else torch.full((rows, vocab), 7.0, dtype=DTYPES[probs], device=dev)
    extra = {} if entries is None else dict(entries=entries.to(dev))
    tokens = draw_tokens(here, coins.to(dev), *on, probs=out, **extra)
    cut = truncate_logits(here, *on, **extra)
    torch.cuda.synchronize()
    tokens, cut = tokens.cpu(), cut.cpu()
    x = logits.float().numpy()
    for r in range(rows):
        i = int(of[r])
        order, mass = ora.kept_part(x[r], float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        want = np.full(vocab, -np.inf, dtype=np.float32)
        want[order] = x[r][order]
        np.testing.assert_array_equal(cut[r].float().numpy(), want, err_msg=f"row {r}")
        flat = coins.view(rows, -1)
        got = [int(v) for v in tokens.view(rows, -1)[r]]
        assert got == [ora.drawn(order, mass, float(c)) for c in flat[r]], f"row {r}"
        if out is not None:
            share = np.zeros(vocab)
            share[order] = mass / mass.sum()
            have = out[r].double().cpu().numpy()
            bound = 1.01 * HALF_STEP[out.dtype] * share + TINY[out.dtype]
            assert (np.abs(have - share) <= bound).all(), f"row {r}"
            assert ((have > 0) <= (share > 0)).all()


RULES = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (1.3, 0, 0.95, 0.0), (0.8, 0, 1.0, 0.05), (0.9, 50, 0.8, 0.02),
         (1.0, 1500, 0.99, 0.0), (1.0, 1500, 1.0, 1e-6), (0.0, 5, 0.5, 0.5)]


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 300, 2049, 50257])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rules_and_sizes(dev, dtype, vocab, rules):
    announce(f"sample rows {dtype} vocab={vocab} rules={rules}")
    _check(dev, _logits(4, vocab, dtype, vocab), *rules, probs="f32")


@pytest.mark.parametrize("dtype,probs", [("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("vocab", [32000, 151936, 1 << 18])
def test_types_at_large_vocabularies(dev, dtype, probs, vocab):
    announce(f"sample rows {dtype} -> {probs} vocab={vocab}")
    t = torch.tensor([0.6, 1.0, 2.0, 5.0])
    k, p = torch.tensor([40, 0, 0, 5000], dtype=torch.int32), torch.tensor([0.95, 0.9, 0.7, 0.999])
    _check(dev, _logits(4, vocab, dtype, 3), t, k, p, 0.0, probs=probs)


def test_mixed_requests_share_a_batch(dev):
    announce("sample rows: entries")
    gen = torch.Generator().manual_seed(5)
    entries = torch.randint(0, 6, (20,), generator=gen)
    t = torch.tensor([0.0, 0.5, 0.8, 1.0, 1.5, 1e-3])
    k = torch.tensor([0, 10, 0, 0, 70, 0], dtype=torch.int32)
    p, m = torch.tensor([1.0, 0.9, 0.5, 1.0, 0.95, 0.9]), torch.tensor([0.0, 0.0, 0.0, 0.3, 0.0, 0.0])
    _check(dev, _logits(20, 5001, "bf16", 9), t, k, p, m, entries=entries, probs="f32",
           coins=torch.rand(20, 64, generator=gen))
    _check(dev, _logits(20, 5001, "bf16", 9), t, k, p, m, entries=entries.int(), coins=torch.rand(20, generator=gen))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [0.0, -3.5])
def test_equal_logits_keep_the_lowest_indices(dev, dtype, value):
    """Rows of one logit: more equals than any list holds, cut by count and by mass."""
    announce(f"sample rows: equal logits {dtype} {value}")
    x = torch.full((6, 40001), value, dtype=DTYPES[dtype])
    x[3, 777] = value + 2
    x[4, ::2] = -torch.inf
    x[5, 1::3] = -0.0
    k = torch.tensor([0, 3000, 0, 3000, 0, 20000], dtype=torch.int32)
    p = torch.tensor([0.5, 1.0, 1.0, 0.75, 0.3, 0.9])
    _check(dev, x, 1.0, k, p, 0.0, probs="f32", coins=torch.tensor([[0.0, 0.31, 0.99999994]]).expand(6, 3).contiguous())


def test_logits_at_the_ends_of_their_type(dev):
    announce("sample rows: ends of the type")
    low = torch.finfo(torch.float32).min
    x = _logits(9, 3001, "f32", 4)
    x[0, 100:] = low
    x[1, 1:] = -torch.inf
    x[2] = -torch.inf
    x[3, 50] = torch.inf
    x[3, 40] = torch.inf
    x[4, 70] = torch.nan
    x[4, 60] = torch.inf
    x[5] = low
    x[6] *= 1e30
    x[7] = torch.where(torch.arange(3001) % 2 == 0, torch.finfo(torch.float32).max, low)
    x[8] *= 1e-30
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    for rules in ((1.0, 0, 0.9, 0.0), (0.5, 2000, 1.0, 0.0), (1.0, 30, 0.99, 0.01), (1e-30, 0, 0.5, 0.0), (float("inf"), 0, 0.5, 0.0)):
        rows = [0, 1, 2, 3, 5, 6, 7, 8]  # (a NaN row is compared below)
        _check(dev, x[rows], *rules, probs="f32")
        t, k, p, m = _rules(1, *rules, dev)
        tokens = draw_tokens(x[4:5].to(dev), torch.full((1, 2), 0.5, device=dev), t, k, p, m)
        assert tokens.tolist() == [[70, 70]]
        cut = truncate_logits(x[4:5].to(dev), t, k, p, m).cpu()
        assert torch.isnan(cut[0, 70]) and int(torch.isneginf(cut).sum()) == 3000


@pytest.mark.parametrize("rules", [(1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, 0, float("nan"), 0.0),
                                   (1.0, -5, 1.0, 0.0), (1.0, 3000, 1.0, 0.0), (1.0, 1 << 30, 1.0, 0.0), (1.0, 0, 1.0, 2.0),
                                   (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, float("nan")), (float("nan"), 9, 0.9, 0.0), (-1.0, 9, 0.9, 0.0)])
def test_rules_at_their_ends(dev, rules):
    announce(f"sample rows: rules {rules}")
    x = _logits(3, 2999, "bf16", 8)
    x[1, 5] = x[1, 900] = x[1, 17] = 30.0  # ties at the top
    _check(dev, x, *rules, probs="f32")


def test_coins_at_their_ends(dev):
    announce("sample rows: coins")
    x = _logits(2, 4099, "f32", 2)
    x[0, :40] = -torch.inf
    coins = torch.tensor([[0.0, 0.99999994, 1.0, 2.0, -1.0, float("nan")]] * 2)
    for rules in ((1.0, 0, 1.0, 0.0), (1.0, 12, 1.0, 0.0)):
        from eagle_harness.vllm.sampling import draw_tokens

        got = draw_tokens(x.to(dev), coins.to(dev), *_rules(2, *rules, dev)).cpu()
        for r in range(2):
            order, mass = ora.kept_part(x[r].numpy(), *rules)
            first, last = int(order[0]), ora.drawn(order, mass, 0.99999994)
            assert got[r, 0] == first and got[r, 1] == last and got[r, 4] == first and got[r, 5] == first
            assert int(got[r, 2]) in order and mass[list(order).index(int(got[r, 2]))] > 0 and got[r, 2] == got[r, 3]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("offset,pad", [(1, 3), (3, 0), (7, 9), (0, 5)])
def test_rows_behind_any_boundary(dev, dtype, offset, pad):
    announce(f"sample rows: {dtype} offset {offset} pad {pad}")
    vocab = 5003

    def place(x):
        store = torch.full((offset + x.shape[0] * (vocab + pad),), 99.0, dtype=x.dtype, device=dev)
        view = store[offset:].view(x.shape[0], vocab + pad)[:, :vocab]
        view.copy_(x)
        return view

    for rules in ((0.8, 30, 0.9, 0.0), (1.5, 0, 0.9, 0.0)):
        _check(dev, _logits(5, vocab, dtype, 1), *rules, probs="f32", place=place)


def test_in_place_and_given_outputs(dev):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce("sample rows: in place, strided outputs, padded rows")
    x = _logits(6, 50257, "bf16", 11).to(dev)
    rules = _rules(6, 0.9, 40, 0.95, 0.0, dev)
    want = truncate_logits(x, *rules)
    store = torch.full((6, 50300), 3.0, dtype=x.dtype, device=dev)
    assert truncate_logits(x, *rules, out=store[:, 9:50266]) is not None
    assert torch.equal(store[:, 9:50266], want) and (store[:, :9] == 3).all() and (store[:, 50266:] == 3).all()
    entries = torch.tensor([0, -1, 2, 6, 1, 5], device=dev)
    y = x.clone()
    assert truncate_logits(y, *rules, entries=entries, out=y) is y
    for r in range(6):
        assert torch.equal(y[r], x[r] if r in (1, 3) else want[r])
    probs = torch.full((6, 50257), -1.0, device=dev)
    draw_tokens(x, torch.rand(6, device=dev), *rules, entries=entries, probs=probs)
    for r in range(6):
        assert bool((probs[r] == -1).all()) == (r in (1, 3))
    # one row for all: an expanded view may be read
    same = truncate_logits(x[:1].expand(6, -1), *rules)
    assert all(torch.equal(same[r], want[0]) for r in range(6))


def test_no_rows(dev):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce("sample rows: no rows")
    x = torch.empty(0, 100, device=dev)
    one = torch.ones(1, device=dev)
    assert draw_tokens(x, torch.empty(0, 2, device=dev), one).shape == (0, 2)
    assert truncate_logits(x, one).shape == (0, 100)


def test_captured_and_on_another_stream(dev):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce("sample rows: graph and stream")
    x = _logits(8, 151936, "bf16", 21).to(dev)
    t = torch.tensor([0.7, 1.0, 1.4, 0.0] * 2, device=dev)
    k = torch.tensor([20, 0, 0, 0] * 2, dtype=torch.int32, device=dev)
    p = torch.tensor([0.9, 0.95, 0.9, 1.0] * 2, device=dev)
    coins = torch.rand(8, 2, device=dev)
    probs, cut = torch.empty(8, 151936, device=dev), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        draw_tokens(x, coins, t, k, p, probs=probs)
        truncate_logits(x, t, k, p, out=cut)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = draw_tokens(x, coins, t, k, p, probs=probs)
        truncate_logits(x, t, k, p, out=cut)
    for seed in range(3):
        x.copy_(_logits(8, 151936, "bf16", 30 + seed))
        coins.copy_(torch.rand(8, 2, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        got = tokens.clone(), probs.clone(), cut.clone()
        again = torch.empty_like(probs)
        assert torch.equal(draw_tokens(x, coins, t, k, p, probs=again), got[0]) and torch.equal(again, got[1])
        assert torch.equal(truncate_logits(x, t, k, p), got[2])
        torch.cuda.synchronize()


def test_truncated_rows_in_the_sampled_walk(dev):
    """Draft children drawn with their probabilities, the target's rows truncated, then the walk: as the oracle's walk over
    rows truncated by the oracle."""
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits
    from eagle_harness.vllm.tree_accept import sample_tree
    from eagle_harness.vllm.verify_layout import TreeStore

    announce("sample rows: with the sampled walk")
    gen = torch.Generator().manual_seed(3)
    reqs, width, vocab = 5, 4, 3000
    parents = np.array([-1, 0, 1, 2], dtype=np.int32)  # chains: row n + 1 drawn from row n
    target = _logits(reqs * width, vocab, "f32", 50)
    guess = target + 0.7 * torch.randn(target.shape, generator=gen)
    t, k, p = torch.full((reqs,), 0.8), torch.full((reqs,), 40, dtype=torch.int32), torch.full((reqs,), 0.9)
    entries = torch.arange(reqs).repeat_interleave(width)
    rules = [v.to(dev) for v in (t, k, p)]
    probs = torch.empty(reqs * width, vocab, device=dev)
    drawn = draw_tokens(guess.to(dev), torch.rand(reqs * width, generator=gen).to(dev), *rules, entries=entries.to(dev), probs=probs)
    drafted = torch.roll(drawn, 1)  # row n holds what its parent's row drew
    cut = truncate_logits(target.to(dev), *rules, entries=entries.to(dev))
    store = TreeStore(reqs, width, dev)
    store.parents[:] = torch.from_numpy(parents).to(dev)
    coins, final = torch.rand(reqs * width, generator=gen), torch.rand(reqs, generator=gen)
    cu = torch.arange(0, reqs * width + 1, width, dtype=torch.int32, device=dev)
    sampled, count = sample_tree(cut, drafted, cu, torch.arange(reqs, dtype=torch.int32, device=dev), store.parents, store,
                                 coins.to(dev), final.to(dev), rules[0], draft_probs=probs)
    torch.cuda.synchronize()
    accepted = 0
    for b in range(reqs):
        rows = slice(b * width, (b + 1) * width)
        want = np.full((width, vocab), -np.inf, dtype=np.float32)
        for j in range(width):
            order, _ = ora.kept_part(target[b * width + j].numpy(), float(t[b]), int(k[b]), float(p[b]))
            want[j, order] = target[b * width + j].numpy()[order]
        tokens, path = ora.walk(want, drafted[rows].cpu().numpy(), parents, coins[rows].numpy(), float(final[b]), float(t[b]),
                                probs[rows].cpu().numpy())
        assert sampled[b, : int(count[b])].tolist() == list(tokens)
        accepted += int(count[b]) - 1
    assert accepted > 0
