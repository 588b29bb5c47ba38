"""Caches and logits whose offsets pass 32 bits: the same small calls, their pages and rows at the far end of allocations of more
than 2^32 bytes (and, at 16 bits, more than 2^31 elements)."""

import pytest
import torch

import test_gpu_kv_pages as kv
import test_gpu_latent_attention as lat
import test_gpu_sample_tree as st
from conftest import announce
from oracle import kv_pages as okv

pytestmark = pytest.mark.gpu

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def far_pages(cache, table, dev, bytes_):
    """``cache`` at the end of one of more than ``bytes_``, and ``table`` with its ids moved there."""
    blocks = cache.shape[0]
    first = bytes_ // (cache[0].numel() * cache.element_size()) + 1
    whole = torch.empty((first + blocks, *cache.shape[1:]), dtype=cache.dtype, device=dev)
    whole[first:] = cache.to(dev)
    return whole, torch.where((table >= 0) & (table < blocks), table + first, table), first


@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_latent_rows(dev, cache):
    announce(f"latent far pages {cache}")
    x = lat.inputs([300, 40, 7], [4, 1, 2], 16, BF16, cache, seed=91)
    want = lat.launch(x, dev)
    whole, table, first = far_pages(x["cache"], x["table"], dev, (1 << 32) + (1 << 30))
    scale = None
    if cache == "fp8":
        scale = torch.cat([torch.ones(first), x["page_scale"]])
    assert torch.equal(lat.launch(x, dev, cache=whole, table=table, page_scale=scale), want)


@pytest.mark.parametrize("heads,dim", [(4, 128), (3, 7)])
def test_pages_written_and_read(dev, heads, dim):
    from eagle_harness.vllm.kv_pages import read_kv_pages

    announce(f"far pages written and read heads {heads} dim {dim}")
    x = kv.batch([5, 0, 30], [9, 20, 3], heads, dim, 16, BF16, seed=92)
    whole, table, first = far_pages(x["cache"].view(torch.uint8), x["table"], dev, (1 << 32) + (1 << 28))
    whole = whole.view(FP8)
    scale = torch.cat([torch.ones(first, heads), x["scale"]]).to(dev)
    kv.write(dict(x, table=table), dev, cache=whole, scale=scale)
    kv.check(x, (whole[first:], scale[first:]))
    starts = torch.tensor([0, 14, 34, 67], dtype=torch.int32)
    out = torch.empty(67, heads, dim, dtype=BF16, device=dev)
    read_kv_pages(whole, None, scale, None, table.to(dev), starts.to(dev), out, None, max_len=40)
    assert torch.equal(out.cpu(), okv.read_pages(whole[first:].cpu(), scale[first:].cpu(), x["table"], starts).to(BF16))


@pytest.mark.parametrize("probs", [None, F32])
def test_rows_of_logits(dev, probs):
    announce(f"sample tree far rows probs {probs}")
    x = st.inputs([6, 3, 8], 8, 1000, BF16, probs, seed=93)
    rows, stride = x["logits"].shape[0], 1 << 27  # 2^31 elements and more
    held = torch.empty(rows * stride, dtype=BF16, device=dev).view(rows, stride)[:, 11:1011]
    held.copy_(x["logits"])
    q = None
    if probs is not None:
        q = torch.empty(rows * (stride >> 1), dtype=probs, device=dev).view(rows, stride >> 1)[:, 5:1005]
        q.copy_(x["q"])
    st.check(x, st.launch(x, dev, held, q))
