"""Padded rows of drawn and truncated batches (entries outside the requests' vectors): what is returned for them is defined, whatever
the memory held that the results are put into."""

import pytest
import torch

import test_gpu_sample_rows as sr
from conftest import announce

pytestmark = pytest.mark.gpu


def _dirty(shape, dtype, value, dev):
    """Leaves memory of this size, filled, to the next tensor of that size."""
    torch.cuda.synchronize()
    torch.full(shape, value, dtype=dtype, device=dev)
    torch.cuda.synchronize()


ENTRIES = [0, -1, 2, 6, 1, 1 << 40, -(1 << 40)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab,offset", [(5, 0), (4999, 3), (50257, 1)])
def test_padded_rows_are_defined(dev, vocab, offset, dtype):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce(f"padded sample rows {dtype} vocab={vocab} offset={offset}")
    rows = len(ENTRIES)
    store = torch.full((offset + rows * (vocab + 5),), 9.0, dtype=sr.DTYPES[dtype], device=dev)
    x = store[offset:].view(rows, vocab + 5)[:, :vocab]
    x.copy_(sr._logits(rows, vocab, dtype, 4))
    entries = torch.tensor(ENTRIES, device=dev)
    rules = sr._rules(6, 0.9, 40, 0.95, 0.0, dev)
    padded = [r for r, e in enumerate(ENTRIES) if not 0 <= e < 6]
    inside = [r for r in range(rows) if r not in padded]
    want = truncate_logits(x[inside], *[v[:len(inside)] for v in rules])
    for draws in (1, 3):
        coins = torch.rand(rows, draws, device=dev)
        _dirty((rows, draws), torch.int64, 123456789, dev)
        tokens = draw_tokens(x, coins, *rules, entries=entries)
        assert (tokens[padded] == 0).all()
        assert torch.equal(tokens[inside], draw_tokens(x[inside], coins[inside], *[v[:len(inside)] for v in rules]))
    _dirty((rows, vocab), x.dtype, 77.0, dev)
    cut = truncate_logits(x, *rules, entries=entries)
    assert torch.equal(cut[padded], x[padded]) and torch.equal(cut[inside], want)


def test_padded_rows_of_large_batches(dev):
    """More rows than are shared by workgroups, and rows of NaN and infinities among the padded."""
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce("padded sample rows: a large batch")
    x = sr._logits(150, 20011, "bf16", 6).to(dev)
    x[7, 5], x[9, 3], x[11] = torch.nan, torch.inf, -torch.inf
    entries = torch.where(torch.arange(150) % 2 == 0, 0, -1).to(dev)
    rules = sr._rules(1, 0.9, 40, 0.95, 0.0, dev)
    _dirty((150, 20011), x.dtype, 77.0, dev)
    cut = truncate_logits(x, *rules, entries=entries)
    assert torch.equal(cut[1::2].view(torch.int16), x[1::2].view(torch.int16))
    _dirty((150,), torch.int64, 123456789, dev)
    tokens = draw_tokens(x, torch.rand(150, device=dev), *rules, entries=entries)
    assert (tokens[1::2] == 0).all() and torch.isneginf(cut[::2]).any(1).all()


def test_a_captured_batch_whose_padding_changes(dev):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce("padded sample rows captured")
    x = sr._logits(6, 32000, "bf16", 2).to(dev)
    coins, rules = torch.rand(6, 2, device=dev), sr._rules(6, 0.9, 40, 0.95, 0.0, dev)
    entries = torch.arange(6, device=dev)
    draw_tokens(x, coins, *rules, entries=entries)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = draw_tokens(x, coins, *rules, entries=entries)
        cut = truncate_logits(x, *rules, entries=entries)
    for live in (6, 3, 5, 1):
        entries.copy_(torch.tensor([r if r < live else -1 for r in range(6)]))
        graph.replay()
        assert (tokens[live:] == 0).all() and torch.equal(cut[live:], x[live:])
        assert torch.equal(tokens[:live], draw_tokens(x[:live], coins[:live], *rules))
        assert torch.equal(cut[:live], truncate_logits(x[:live], *rules))
