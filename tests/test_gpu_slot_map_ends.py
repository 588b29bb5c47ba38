"""Slots of the rows that no request has: before the first request's rows as behind the last one's."""

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [0, 1, 5, 3000, 70000])
@pytest.mark.parametrize("first", [0, 1, 700, 5000])
def test_rows_that_no_request_has(dev, first, rows):
    from eagle_harness.vllm.page_tables import slot_maps

    announce(f"slots: {rows} rows, the first request's from {first} on")
    i32 = dict(dtype=torch.int32, device=dev)
    table, pages = torch.arange(40, **i32).view(4, 10), torch.tensor([10, 3, 0, 7], **i32)
    starts = torch.tensor([first, first + 3, first + 3, first + 9], **i32)
    slots = torch.full((rows,), 77, dtype=torch.int64, device=dev)
    slot_maps(table, pages, torch.tensor([3, 0, 1], **i32), torch.tensor([0, 5, 17], **i32), starts, 16, slots=slots)
    want = torch.full((first + 9 + max(rows, 9),), -1, dtype=torch.int64)
    want[first : first + 3] = 30 * 16 + torch.arange(3)
    want[first + 3 : first + 9] = 11 * 16 + 1 + torch.arange(6)
    assert torch.equal(slots.cpu(), want[:rows])
