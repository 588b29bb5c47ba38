"""Draft rows over fp8 pages behind the end of their page table (an extend padded past it, a length beyond it): they see the keys of
their window that the table has, and none twice. The bound is that of ``test_gpu_row_attention_fp8.py``."""

import pytest
import torch

import test_gpu_row_attention_fp8 as rows
from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 1, 3, 40])
@pytest.mark.parametrize("step,length", [(0, 94), (0, 96), (0, 99), (0, 200), (2, 97), (2, 130)])
def test_rows_behind_the_table(dev, step, length, window, dtype):
    announce(f"fp8 rows behind the table: length={length} step={step} window={window} {dtype}")
    gen = torch.Generator().manual_seed(length + window)
    page, hkv, dim, n, hq = 16, 2, 64, 5, 4
    room = 6 * page
    keys, ks = rows._cache(gen, 9, page, hkv, dim)
    values, vs = rows._cache(gen, 9, page, hkv, dim)
    table, seq = torch.randperm(9, generator=gen)[:6].view(1, 6).int(), torch.tensor([length])
    anc = torch.randint(0, 9 * page, (1, n, step), generator=gen).int() if step else None
    q = torch.randn(n, hq, dim, generator=gen).to(dtype)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = rows._launch(dev, *[on(t) for t in (q, keys, values, ks, vs, table, seq, anc)], rows=n, step=step, window=window, splits=3,
                       table_page=page).cpu().double()
    wide_k, wide_v = rows._wide(keys, ks).view(-1, hkv, dim), rows._wide(values, vs).view(-1, hkv, dim)
    e = rows.STEP[dtype]
    for t in range(n):
        newest = length - 1 if step else length + t
        at = torch.arange(max(newest - window + 1, 0) if window else 0, min(newest + 1, room)) if newest - window + 1 < room or not window \
            else torch.arange(0)
        slots = table[0, at // page].long() * page + at % page
        if step:
            slots = torch.cat([slots, anc[0, t].long()])
        if not len(slots):
            assert (got[t] == 0).all()
            continue
        for h in range(hq):
            k, v = wide_k[slots, h // 2], wide_v[slots, h // 2]
            w = torch.softmax(k @ q[t, h].double() * dim**-0.5, 0)
            want = w @ v
            bound = (e + 2.0**-16) * (w @ v.abs()) + e * want.abs() + 2.0**-25
            assert ((got[t, h] - want).abs() <= bound).all(), (t, h)


def test_no_requests(dev):
    announce("fp8 rows: no requests")
    cache, scales = torch.zeros(4, 16, 2, 64, device=dev).to(torch.float8_e4m3fn), torch.ones(4, 2, device=dev)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    got = rows._launch(dev, q, cache, cache, scales, scales, none.view(0, 6), none, None, rows=2, step=0, window=0, splits=2, table_page=16)
    assert got.shape == q.shape
