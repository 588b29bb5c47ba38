"""Weights of draft rows over fp8 pages where pages without values (scale 0, as ``write_kv_pages`` leaves a page of zeros, or
codes of zeros) stand beside pages of small values: the empty pages' keys take their share of the softmax, and the other
weights keep their bits, however far the value scales lie apart. The bound is that of ``test_gpu_row_attention_fp8.py``."""

import pytest
import torch

import test_gpu_row_attention_fp8 as rows
from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("empty", ["scale", "codes"])
@pytest.mark.parametrize("dim,hq,n", [(64, 8, 4), (128, 4, 1), (128, 32, 4), (256, 24, 2)])
@pytest.mark.parametrize("size,lift", [(-9, 10), (-14, 6), (-17, 10), (-20, 0)])
def test_pages_without_values_beside_small_ones(dev, size, lift, dim, hq, n, empty, dtype):
    """Value scales of 2^size; the keys of the empty pages score 2^lift above the others'."""
    announce(f"fp8 rows: empty pages by {empty}, values 2^{size}, lift {lift}, {hq}x{dim} {dtype}")
    gen = torch.Generator().manual_seed(dim + lift)
    page, pages, hkv = 16, 10, 2
    keys, ks = rows._cache(gen, pages, page, hkv, dim, 0.1)
    values = (100 * torch.randn(pages, page, hkv, dim, generator=gen)).clamp(-448, 448)
    vs = torch.full((pages, hkv), 2.0**size)
    at = [1, 7]
    values[at] = 0
    vs[at] = 0.0 if empty == "scale" else 1.0
    values = values.to(torch.float8_e4m3fn)
    # a row's first element is 4, and an empty page's key has nothing but its own: `lift` powers of two; the others' is 0
    wide = keys.float()
    wide[..., 0] = 0
    wide[at] = 0
    wide[at, :, :, 0] = 448
    ks[at] = lift * 0.6931471805599453 * dim**0.5 / 4 / 448
    keys = wide.to(torch.float8_e4m3fn)
    q = torch.randn(n, hq, dim, generator=gen)
    q[..., 0] = 4
    q = q.to(dtype)
    table, seq = torch.randperm(pages, generator=gen).view(1, -1).int(), torch.tensor([pages * page - n])
    args = [t.to(dev) for t in (q, keys, values, ks, vs, table, seq)]
    got = rows._launch(dev, *args, None, rows=n, step=0, window=0, splits=2, table_page=page)
    rows._compare(got, q, rows._wide(keys, ks), rows._wide(values, vs), table, seq, None, rows_per_request=n, step=0, window=0,
                  table_page=page)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pages_of_zeros_alone(dev, dtype):
    """Nothing but pages without values: zeros, not NaN."""
    announce(f"fp8 rows: zeros alone {dtype}")
    gen = torch.Generator().manual_seed(1)
    keys, ks = rows._cache(gen, 6, 16, 2, 128, 0.1)
    values, vs = torch.zeros_like(keys), torch.zeros(6, 2)
    table, seq = torch.arange(6).view(1, 6).int(), torch.tensor([90])
    q = torch.randn(3, 8, 128, generator=gen).to(dtype)
    got = rows._launch(dev, *[t.to(dev) for t in (q, keys, values, ks, vs, table, seq)], None, rows=3, step=0, window=0, splits=2,
                       table_page=16)
    assert (got == 0).all()


@pytest.mark.parametrize("dim,hq", [(64, 4), (128, 32), (256, 12)])
@pytest.mark.parametrize("bad", [5, 66, 97])
def test_nan_codes_under_fp16_rows(dev, bad, dim, hq):
    """A NaN code among the values of position 5 or 66 (rows at 95 to 98 see both) or of 97, which rows 2 and 3 alone see."""
    announce(f"fp8 rows: NaN at {bad} under fp16 rows of {dim}")
    gen = torch.Generator().manual_seed(dim)
    page, hkv, n = 16, 2, 4
    keys, ks = rows._cache(gen, 7, page, hkv, dim, 0.2)
    values, vs = rows._cache(gen, 7, page, hkv, dim, 0.2)
    table, seq = torch.arange(7).view(1, 7).int(), torch.tensor([95])
    q = torch.randn(n, hq, dim, generator=gen).to(torch.float16)
    run = lambda: rows._launch(dev, *[t.to(dev) for t in (q, keys, values, ks, vs, table, seq)], None, rows=n, step=0, window=0,  # noqa: E731
                               splits=2, table_page=page).cpu()
    want = run()
    values.view(torch.uint8)[bad // page, bad % page, 0, 33] = 0x7F
    want[2 if bad == 97 else 0 :, : hq // 2, 33] = torch.nan
    assert torch.equal(run().nan_to_num(99.0), want.nan_to_num(99.0))
