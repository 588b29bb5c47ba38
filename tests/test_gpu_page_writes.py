"""Page writes at what a batch holds beside ordinary rows: padded requests, path entries of no row."""

import pytest
import torch

import test_gpu_kv_pages as kv
from conftest import announce

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("heads,dim,page", [(4, 256, 16), (3, 7, 5), (2, 264, 40)])
def test_paths_that_name_no_row_leave_pages_and_scales(dev, heads, dim, page):
    """A request padded into the batch (no rows, another's slot), and paths whose last page's entries name none."""
    announce(f"write pages of no path row heads {heads} dim {dim} page {page}")
    x = kv.batch([0, page - 2, 3 * page, 0], [0, 6, 4, 5], heads, dim, page, BF16, seed=61)
    path = torch.tensor([[0, 1, 3, 2, 0, 0], [1, 4, 9, 7, -2, 6], [8, 9, -1, 4, 5, 6]], dtype=torch.int32)
    path_len, slots = torch.tensor([4, 6, 6], dtype=torch.int32), torch.tensor([0, 1, 2, 2])
    got = kv.write(x, dev, idx_mapping=slots.to(dev), path=path.to(dev), path_len=path_len.to(dev))
    kv.check(x, got, path=path, path_len=path_len, slots=slots)
    touched = int(x["table"][1, 0])  # of request 1 the first page's two rows alone
    rest = [p for p in range(x["blocks"]) if p != touched and p not in x["table"][3].tolist()]
    assert torch.equal(got[1].cpu()[rest], x["scale"][rest]) and kv.same(got[0][rest], x["cache"][rest])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,dim,page", [(4, 256, 16), (3, 7, 5), (2, 264, 40)])
def test_pages_of_infinities_and_zeros_read_back_saturated(dev, dtype, heads, dim, page):
    from eagle_harness.vllm.kv_pages import read_kv_pages

    announce(f"write pages of infinities heads {heads} dim {dim} page {page} {dtype}")
    n = 2 * page + 1
    x = kv.batch([0, 3], [n, 1], heads, dim, page, dtype, seed=62)
    x["key"][:] = 0.0
    x["key"][1, :, 2], x["key"][page - 1, 0, dim - 1], x["key"][page, 1, 0] = float("inf"), -float("inf"), float("inf")
    x["key"][n, 0, 1] = float("inf")  # of the request behind three positions
    x["scale"][int(x["table"][1, 0])] = 0.0
    x["scale"][int(x["table"][1, 0]), 0] = 0.5
    got = kv.write(x, dev)
    kv.check(x, got)
    out = torch.empty(n, heads, dim, device=dev)
    read_kv_pages(got[0], None, got[1], None, x["table"].to(dev), torch.tensor([0, n], device=dev), out, None, max_len=n)
    assert torch.equal(out.cpu(), x["key"][:n].float().clamp(-448.0, 448.0))
    assert float(got[1][int(x["table"][1, 0]), 0]) == 0.5
