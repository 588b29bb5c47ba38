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


def test_infinities_alone_saturate_and_do_not_become_zeros():
    cache, scale = pages(dim=4)
    inf, nan = float("inf"), float("nan")
    key = torch.zeros(3, 2, 4)
    key[0, 0, 1], key[1, 0, 2] = inf, -inf
    key[2, 1, 0] = nan  # head 1: no infinity, a scale of 0
    okv.write_pages(key, cache, scale, torch.tensor([[1, 2]]), torch.tensor([0]), torch.tensor([0, 3]))
    got = okv.read_pages(cache, scale, torch.tensor([[1, 2]]), torch.tensor([0, 3]))
    want = torch.zeros(3, 2, 4, dtype=torch.float64)
    want[0, 0, 1], want[1, 0, 2], want[2, 1, 0] = 448.0, -448.0, nan
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and scale[1].tolist() == [1.0, 0.0]
    # behind positions that have a scale, that one stays
    scale[1] = 0.25
    okv.write_pages(key[:1], cache, scale, torch.tensor([[1, 2]]), torch.tensor([3]), torch.tensor([0, 1]))
    assert scale[1].tolist() == [0.25, 0.25] and float(cache[1, 3, 0, 1]) == 448.0
