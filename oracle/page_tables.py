"""Page tables, request by request, on lists: what ``resize_tables`` and ``slot_maps`` leave."""

from __future__ import annotations


def resized(table, pages, idx, lens, stack, capacity, page):
    """``table`` (lists of pages a slot), ``pages`` and ``stack`` (the free ones) in place."""
    slots, most = len(table), len(table[0])
    if len(stack) + sum(max(0, pages[s] - -(-max(n, 0) // page)) for s, n in zip(idx, lens) if 0 <= s < slots) > capacity:
        return
    for s, n in reversed(list(zip(idx, lens))):
        need = -(-max(n, 0) // page)
        if 0 <= s < slots and need < pages[s]:
            stack.extend(table[s][at] for at in range(pages[s] - 1, need - 1, -1))
            pages[s] = need
    wanted, there = 0, len(stack)
    for s, n in zip(idx, lens):
        need = -(-max(n, 0) // page)
        if not 0 <= s < slots or not pages[s] < need <= most:
            continue
        wanted += need - pages[s]
        if wanted > there:
            continue
        while pages[s] < need:
            table[s][pages[s]] = stack.pop()
            pages[s] += 1


def slot_of(table, pages, s, position, page):
    if not 0 <= s < len(table) or not 0 <= position < pages[s] * page:
        return -1
    return table[s][position // page] * page + position % page
