"""Draft rows over fp8 pages in many splits: more partials than one run of the merge takes, and more than four of them do. How many
were used is counted in the scratch, which holds NaN before the call. The bound is that of ``test_gpu_row_attention_fp8.py``."""

import pytest
import torch

import test_gpu_row_attention_fp8 as rows
from conftest import announce

pytestmark = pytest.mark.gpu


def _run(dev, seed, bs, n, step, hq, hkv, dim, dtype, window, lens, width, splits, page=16):
    """Returns how many partials a row had."""
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention, rows_padded

    gen = torch.Generator().manual_seed(seed)
    need = -(-(max(lens) + n * max(step, 1)) // page)
    pages = bs * need + 3
    keys, ks = rows._cache(gen, pages, page, hkv, dim)
    values, vs = rows._cache(gen, pages, page, hkv, dim)
    table = torch.zeros(bs, width, dtype=torch.int32)
    table[:, :need] = torch.randperm(pages, generator=gen)[: bs * need].view(bs, need)
    seq = torch.tensor(lens)
    q = torch.randn(bs * n, hq, dim, generator=gen).to(dtype)
    anc = None
    if step:
        at = seq[:, None, None] + torch.randint(0, n * step, (bs, n, step), generator=gen)
        anc = (table[torch.arange(bs)[:, None, None], at // page] * page + at % page).int()
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    parts = bs * hq * (splits + 1) * rows_padded(n)
    part, lse = torch.full((parts, dim), torch.nan, device=dev), torch.full((parts,), torch.nan, device=dev)
    got = torch.full_like(q, 5.0, device=dev)
    rows_attention(on(q), on(keys), on(values), got, part, lse, on(table), on(seq), on(anc), rows_per_request=n, step=step, window=window,
                   scale=dim**-0.5, launch=RowsLaunch(splits=splits, block_n=32), table_page=page, k_scale=on(ks), v_scale=on(vs))
    torch.cuda.synchronize()
    rows._compare(got, q, rows._wide(keys, ks), rows._wide(values, vs), table, seq, anc, rows_per_request=n, step=step, window=window,
                  table_page=page)
    used = (~torch.isnan(lse)).view(bs, hq, splits + 1, rows_padded(n))[..., :n].sum(2)
    assert (used == used[0, 0, 0]).all()
    return int(used[0, 0, 0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [0, 2])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (4, 1, 128), (6, 1, 256)])
def test_long_contexts(dev, hq, hkv, dim, step, dtype):
    announce(f"fp8 rows: long contexts {hq}/{hkv}x{dim} step={step} {dtype}")
    for length, least in ((4096, 9), (12000, 33)):
        used = _run(dev, length + dim, 1, 2, step, hq, hkv, dim, dtype, 0, [length], length // 16 + 1, 64)
        assert used >= least, used


@pytest.mark.parametrize("step", [0, 3])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows_inside_long_contexts(dev, dim, step):
    """The window leaves the first half of the context out; and a few keys in a table of many pages, where most splits are empty."""
    announce(f"fp8 rows: windows of many splits {dim} step={step}")
    assert _run(dev, 3, 1, 3, step, 8, 2, dim, torch.bfloat16, 5001, [11000], 700, 64) >= 9
    for lens in ([1, 300], [0, 31]):
        assert _run(dev, 4, 2, 3, step, 8, 2, dim, torch.bfloat16, 0, lens, 700, 64) >= 33
