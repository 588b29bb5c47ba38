"""The oracle of the page tables: a negative length holds no pages, and gives back no more than are held."""

import pytest

from oracle.page_tables import resized


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("length", [0, -1, -40])
def test_a_negative_length_gives_back_what_is_held(page, length):
    table, pages, stack = [[4, 2, 0], [1, 0, 0]], [2, 1], [3, 0]
    resized(table, pages, [0, 1], [length, page], stack, 5, page)
    assert pages == [0, 1] and stack == [3, 0, 2, 4]
