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


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,part", [(128, 128), (96, 64), (20, 6)])
def test_heads_beside_the_rotated_ones(dev, dim, part, interleaved):
    """The parts of one packed projection, rotated into other parts of it."""
    from eagle_harness.vllm.rotary import rotary_frequencies, rotate_rows

    announce(f"rotated beside the inputs {part} of {dim} interleaved={interleaved}")
    gen = torch.Generator().manual_seed(dim)
    packed = torch.randn(37, 12, dim, generator=gen).bfloat16().to(dev)
    k_out = torch.empty(37, 2, dim, dtype=packed.dtype, device=dev)
    before, at, f = packed.clone(), torch.arange(37, device=dev) * 1001, rotary_frequencies(part, device=dev)[0]
    rotate_rows(packed[:, 0:4], packed[:, 4:6], at, f, interleaved=interleaved, q_out=packed[:, 7:11], k_out=k_out)
    q, k = rotate_rows(before[:, 0:4].clone(), before[:, 4:6].clone(), at, f, interleaved=interleaved)
    assert torch.equal(packed[:, 7:11], q) and torch.equal(k_out, k)
    assert torch.equal(packed[:, :7], before[:, :7]) and torch.equal(packed[:, 11:], before[:, 11:])


def test_a_batch_table_beside_the_block_table(dev):
    from eagle_harness.vllm.page_tables import slot_maps

    announce("a batch table beside the block table")
    i32 = dict(dtype=torch.int32, device=dev)
    wide = torch.full((6, 21), -7, **i32)
    table, batch = wide[:, :10], wide[:3, 10:20]
    table.copy_(torch.arange(60, **i32).view(6, 10))
    before, pages = table.clone(), torch.tensor([10, 3, 0, 7, 1, 5], **i32)
    idx, context, starts = torch.tensor([3, 0, 2], **i32), torch.tensor([100, 20, 0], **i32), torch.tensor([0, 9, 19, 22], **i32)
    got = slot_maps(table, pages, idx, context, starts, 16, slots=torch.empty(25, dtype=torch.int64, device=dev), batch_table=batch)
    want = slot_maps(before, pages, idx, context, starts, 16, slots=torch.empty(25, dtype=torch.int64, device=dev),
                     batch_table=torch.empty(3, 10, **i32))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(table, before)
    assert (wide[:, 20] == -7).all() and (wide[3:, 10:] == -7).all()
