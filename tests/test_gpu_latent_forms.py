"""Latent verify attention at the ends of its caches and schedules."""

import pytest
import torch

import test_gpu_latent_attention as lat
from conftest import announce

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
