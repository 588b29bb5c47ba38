"""Outputs that lie beside the inputs in one wider store: what they are in stores of their own, and nothing else is written."""

import pytest
import torch

import test_gpu_sample_rows as sr
from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [4099, 32000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_columns_beside_the_logits(dev, dtype, vocab):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    announce(f"outputs beside the logits {dtype} vocab={vocab}")
    rows = 5
    wide = torch.full((rows, 2 * vocab + 3), 9.0, dtype=sr.DTYPES[dtype], device=dev)
    x, beside = wide[:, 1 : vocab + 1], wide[:, vocab + 1 : 2 * vocab + 1]
    x.copy_(sr._logits(rows, vocab, dtype, 3))
    alone, coins = x.clone(), torch.rand(rows, 2, device=dev)
    for rules in ((0.8, 30, 0.9, 0.0), (1.0, 0, 1.0, 0.0)):
        rules = sr._rules(rows, *rules, dev)
        probs = torch.empty_like(alone)
        want = draw_tokens(alone, coins, *rules, probs=probs)
        assert torch.equal(draw_tokens(x, coins, *rules, probs=beside), want) and torch.equal(beside, probs)
        assert truncate_logits(x, *rules, out=beside) is beside
        assert torch.equal(beside, truncate_logits(alone, *rules)) and torch.equal(x, alone)
        assert (wide[:, :1] == 9).all() and (wide[:, 2 * vocab + 1 :] == 9).all()
