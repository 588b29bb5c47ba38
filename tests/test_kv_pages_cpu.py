"""The fp8 page oracle on the CPU: which pages a round's writes touch, and what infinities become."""

import torch

from oracle import kv_pages as okv

FP8 = torch.float8_e4m3fn


def pages(blocks=4, page=4, heads=2, dim=3):
    cache = torch.full((blocks, page, heads, dim), 2.0).to(FP8)
    return cache, torch.full((blocks, heads), 0.5)


def test_a_path_that_names_no_row_leaves_pages_and_scales():
    """A request padded into a batch: no rows, a slot of the store whose path is another request's."""
    cache, scale = pages()
    key = torch.ones(2, 2, 3)
    path = torch.tensor([[0, 1, 0, 0], [5, -3, 9, 0]])
    for starts, slots in (([0, 0], [0]), ([0, 2], [1])):
        got, factor = cache.clone(), scale.clone()
        okv.write_pages(key, got, factor, torch.tensor([[1, 2]]), torch.tensor([0]), torch.tensor(starts), path=path,
                        path_len=torch.tensor([2, 3]), slots=torch.tensor(slots))
        assert torch.equal(factor, scale) and torch.equal(got.view(torch.uint8), cache.view(torch.uint8))
