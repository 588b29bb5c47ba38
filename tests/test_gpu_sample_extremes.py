"""Tree acceptance by sampling where maxima are large or temperatures small: rows and whole pieces of rows masked by a lowest
value, temperatures down to the smallest, against the 64-bit oracle token for token."""

import pytest
import torch

import test_gpu_sample_tree as st
from conftest import announce

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF16, None), (F16, None), (F32, None), (BF16, F32), (F32, F32), (F32, BF16)]


def masks(dtype):
    return [torch.finfo(dtype).min, -3e4 if dtype == F16 else -1e30, -float("inf")]


@pytest.mark.parametrize("dtype,probs", TYPES)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_pieces_that_are_all_masked(dev, dtype, probs, which):
    """Every token of a vocabulary's end, of its middle and of all but its end masked: pieces with no ordinary logit."""
    announce(f"sample tree masked pieces {dtype} probs {probs} mask {which}")
    x = st.inputs([6] * 8, 6, 12288, dtype, probs, seed=50)
    low = masks(dtype)[which]
    x["temperature"] = torch.tensor([1.0, 0.7, 0.35, 1.3, 0.9, 0.11, 3.0, 0.5])
    for b in range(8):
        lo, hi = [(8192, 12288), (4096, 8192), (0, 8192), (100, 12288)][b % 4]
        rows = slice(6 * b, 6 * b + 6)
        held = x["logits"][rows, lo:hi].clone()
        x["logits"][rows, lo:hi] = low
        if b >= 4:  # the drafted tokens stay likely, among their masked neighbours
            x["logits"][rows, lo:hi] = torch.where(held > 4, held, x["logits"][rows, lo:hi])
    st.check(x, st.launch(x, dev))


@pytest.mark.parametrize("dtype,probs", TYPES)
@pytest.mark.parametrize("vocab", [90, 5000, 9000])
def test_rows_that_are_all_masked_are_uniform(dev, dtype, probs, vocab):
    announce(f"sample tree lowest rows {dtype} probs {probs} vocab {vocab}")
    x = st.inputs([4] * 8, 4, vocab, dtype, probs, seed=51)
    x["logits"][:] = torch.finfo(dtype).min
    x["logits"][20:] = torch.finfo(dtype).max
    x["temperature"] = torch.tensor([1.0, 0.7, 0.35, 1.3, 1.0, 0.7, 1e-3, 2.0])
    # the middle of a token's share of the running sum
    x["final"] = (torch.tensor([0, vocab // 2, vocab - 1, vocab // 3, vocab // 7, vocab // 2, vocab // 5, vocab - 2]) + 0.5) / vocab
    x["coins"][:] = 0.99  # a share of 1 / vocab, or q times the row's mass: rejected, but for draws of a peaked q
    if probs is not None:
        x["q"][:] = 1.0 / vocab
        x["coins"][:] = 0.0
        x["coins"][3::4] = 0.999
    st.check(x, st.launch(x, dev))


@pytest.mark.parametrize("dtype,probs", TYPES)
@pytest.mark.parametrize("vocab", [90, 9000])
def test_temperatures_near_zero_are_the_argmax(dev, dtype, probs, vocab):
    announce(f"sample tree small temperatures {dtype} probs {probs} vocab {vocab}")
    x = st.inputs([6] * 8, 6, vocab, dtype, probs, seed=52)
    x["temperature"] = torch.tensor([1e-6, 1e-12, 1e-15, 1e-18, 1e-20, 1e-30, 1e-38, 1e-45])
    assert bool((x["temperature"] > 0).all())
    x["logits"][::2] -= 37.0  # maxima of either sign
    st.check(x, st.launch(x, dev))


@pytest.mark.parametrize("dtype,probs", TYPES)
def test_logits_far_from_zero(dev, dtype, probs):
    """A constant on a row changes nothing: maxima at a thousandth of the type's range, differences of ordinary size."""
    announce(f"sample tree far logits {dtype} probs {probs}")
    x = st.inputs([6] * 4, 6, 9000, F32, probs, seed=53)
    far = torch.finfo(dtype).max / 1024
    step = torch.finfo(dtype).eps * far * 2  # of the type's grid there
    x["logits"] = ((x["logits"] * 4).round() * step + torch.tensor([far, -far]).repeat(12)[:, None]).to(dtype)
    x["temperature"] = torch.full((4,), step * 4.0)
    st.check(x, st.launch(x, dev))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("probs", [None, F32])
def test_a_coin_on_the_border_of_two_pieces(dev, dtype, probs):
    """Rows whose second half repeats the first, and a final coin of a half: the running sum reaches it exactly where a piece
    ends, and the next token is the first one past it (or, by the sums' rounding, the last one before)."""
    announce(f"sample tree border {dtype} probs {probs}")
    n, vocab = 96, 16384
    x = st.inputs([1] * n, 1, vocab, dtype, probs, seed=54)
    half = torch.randn(n, vocab // 2, generator=torch.Generator().manual_seed(54)).to(dtype)
    x["logits"] = torch.cat([half, half], 1)
    x["final"][:] = 0.5
    x["temperature"][:] = 1.0
    sampled, count, _ = st.launch(x, dev)
    assert count.tolist() == [1] * n
    assert {int(t) for t in sampled[:, 0].cpu()} <= {vocab // 2 - 1, vocab // 2}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("probs", [None, F32])
def test_a_coin_on_the_border_of_two_halves_with_masked_tokens_between(dev, dtype, probs):
    """As above within a piece: the second half begins with eight tokens that may not be drawn."""
    announce(f"sample tree border and masks {dtype} probs {probs}")
    n, vocab = 256, 512
    x = st.inputs([1] * n, 1, vocab, dtype, probs, seed=55)
    half = torch.randn(n, vocab // 2, generator=torch.Generator().manual_seed(55)).to(dtype)
    half[:, :8] = -float("inf")
    x["logits"] = torch.cat([half, half], 1)
    x["final"][:] = 0.5
    x["temperature"][:] = 1.0
    sampled, count, _ = st.launch(x, dev)
    assert count.tolist() == [1] * n
    assert {int(t) for t in sampled[:, 0].cpu()} <= {vocab // 2 - 1, vocab // 2 + 8}
