"""Batches of more rows than are shared by workgroups (from 129 on one writes a whole row): against the oracle, and bit for bit
what the same rows give in small batches."""

import pytest
import torch

import test_gpu_sample_rows as sr
from conftest import announce

pytestmark = pytest.mark.gpu

# greedy, lists by top-k, by min-p and by top-p, rows that keep much or all, cuts inside the bins
T = torch.tensor([0.0, 0.7, 1.0, 0.8, 1.3, 1.0, 1.0, 2.5])
K = torch.tensor([0, 20, 0, 0, 0, 0, 3000, 0], dtype=torch.int32)
P = torch.tensor([1.0, 0.9, 1.0, 0.95, 0.9, 1.0, 0.99, 0.8])
M = torch.tensor([0.0, 0.0, 0.05, 0.0, 0.0, 0.0, 0.0, 1e-5])


@pytest.mark.parametrize("dtype,probs", [("bf16", "f32"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("rows", [127, 128, 129])
def test_batches_around_the_shared_ones(dev, rows, dtype, probs):
    announce(f"sample batches: {rows} rows {dtype} -> {probs}")
    entries = torch.arange(rows) % 8
    x = sr._logits(rows, 20011, dtype, rows)
    coins = torch.rand(rows, 2, generator=torch.Generator().manual_seed(rows))
    sr._check(dev, x, T, K, P, M, coins=coins, probs=probs, entries=entries)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(256, 50257), (131, 151936)])
def test_large_batches_are_their_rows(dev, rows, vocab, dtype):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce(f"sample batches: {rows} x {vocab} {dtype} against small ones")
    x, rules = sr._logits(rows, vocab, dtype, 5).to(dev), [v.to(dev) for v in (T, K, P, M)]
    entries, coins = (torch.arange(rows) * 5 % 8).to(dev), torch.rand(rows, 2, device=dev)
    probs = torch.full((rows, vocab), 7.0, device=dev)
    tokens, cut = draw_tokens(x, coins, *rules, entries=entries, probs=probs), truncate_logits(x, *rules, entries=entries)
    same = x.clone()
    assert torch.equal(truncate_logits(same, *rules, entries=entries, out=same), cut)
    few = torch.empty(16, vocab, device=dev)
    for r in range(0, rows, 16):
        part = slice(r, min(r + 16, rows))
        out = few[: part.stop - r]
        assert torch.equal(draw_tokens(x[part], coins[part], *rules, entries=entries[part], probs=out), tokens[part])
        assert torch.equal(out, probs[part])
        assert torch.equal(truncate_logits(x[part], *rules, entries=entries[part]), cut[part])
    sr._check(dev, x[-9:].cpu(), T, K, P, M, coins=coins[-9:].cpu(), probs="f32", entries=entries[-9:].cpu())
