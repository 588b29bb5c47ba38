"""Draft-row attention over fp8 pages on the GPU against the oracle on the dequantized caches, in 64 bits.

Error: the weights are rounded to the rows' 16 bits (half a step e: 2^-8 bf16, 2^-11 fp16), the output once more; scores,
exponentials and sums are in 32 bits (scores of up to 30 or so in the log2 domain: 30 * 2^-24 relative in a weight, taken as
2^-16). So |got - want| <= (e + 2^-16) sum w |v| / sum w, plus e |want|, which the oracle gives by its run on |v|."""

import pytest
import torch

from conftest import announce
from oracle import row_attention as ora

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _quantized(x, scale):
    return (x / scale[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)


def _cache(gen, pages, page, heads, dim, spread=1.0):
    x = torch.randn(pages, page, heads, dim, generator=gen) * torch.exp(spread * torch.randn(pages, 1, heads, 1, generator=gen))
    scale = x.abs().amax((1, 3)) / 448
    return _quantized(x, scale), scale


def _wide(cache, scale):
    return cache.float().double() * scale.double()[:, None, :, None]


def _launch(dev, q, keys, values, ks, vs, table, seq, anc, *, rows, step, window, splits, table_rows=None, table_page, out=None):
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention, rows_padded

    bs, heads, dim = q.shape[0] // rows, q.shape[1], q.shape[2]
    n = bs * heads * (splits + 1) * rows_padded(rows)
    out = torch.full_like(q, 5.0) if out is None else out
    part, lse = torch.full((n, dim), torch.nan, device=dev), torch.full((n,), torch.nan, device=dev)
    rows_attention(q, keys, values, out, part, lse, table, seq, anc, rows_per_request=rows, step=step, window=window, scale=dim**-0.5,
                   launch=RowsLaunch(splits=splits, block_n=32), table_rows=table_rows, table_page=table_page, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    return out


def _compare(got, q, k, v, table, seq, anc, **kw):
    """``k``, ``v``: the caches in 64 bits."""
    args = dict(scale=q.shape[-1] ** -0.5, **kw)
    wide = q.double()
    want = ora.rows_attention(wide, k, v, table, seq, anc, **args)
    size = ora.rows_attention(wide, k, v.abs(), table, seq, anc, **args)
    e = STEP[got.dtype]
    bound = (e + 2.0**-16) * size + e * want.abs() + 2.0**-25
    far = (got.cpu().double() - want).abs()
    assert (far <= bound).all(), float((far - bound).max())


def _case(dev, seed, bs, rows, step, hq, hkv, dim, dtype, window, low, high, page, splits, spread=1.0, table_page=None):
    gen = torch.Generator().manual_seed(seed)
    width = -(-(high + rows * max(step, 1)) // page) + 1
    pages = bs * width + 3
    keys, ks = _cache(gen, pages, page, hkv, dim, spread)
    values, vs = _cache(gen, pages, page, hkv, dim, spread)
    table = torch.randperm(pages, generator=gen)[: bs * width].view(bs, width).int()
    seq = torch.randint(low, high + 1, (bs,), generator=gen)
    q = torch.randn(bs * rows, hq, dim, generator=gen).to(dtype)
    req = torch.randperm(bs, generator=gen)
    anc = None
    if step:
        at = seq[:, None, None] + torch.randint(0, rows * step, (bs, rows, step), generator=gen)
        anc = (table[req][torch.arange(bs)[:, None, None], at // page] * page + at % page).int()
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = _launch(dev, on(q), on(keys), on(values), on(ks), on(vs), on(table), on(seq), on(anc), rows=rows, step=step, window=window,
                  splits=splits, table_rows=on(req), table_page=page)
    _compare(got, q, _wide(keys, ks), _wide(values, vs), table, seq, anc, rows_per_request=rows, step=step, window=window,
             table_rows=req, table_page=page)


HEADS = [(8, 2, 64), (4, 4, 128), (8, 2, 128), (6, 1, 256), (12, 2, 256), (40, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim", HEADS)
@pytest.mark.parametrize("step,rows", [(1, 1), (3, 4), (11, 8), (0, 1), (0, 5), (0, 16)])
def test_steps_and_heads(dev, step, rows, hq, hkv, dim, dtype):
    announce(f"fp8 rows step={step} rows={rows} heads={hq}/{hkv}x{dim} {dtype}")
    _case(dev, step * 10 + rows, 2, rows, step, hq, hkv, dim, dtype, 0, 30, 200, 16, 3)


@pytest.mark.parametrize("window", [0, 1, 7, 33, 96, 500])
@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("step,rows", [(2, 3), (0, 6)])
def test_windows_and_pages(dev, step, rows, page, window):
    announce(f"fp8 rows window={window} page={page} step={step}")
    _case(dev, window + page, 3, rows, step, 8, 2, 64, torch.bfloat16, window, 1, 300, page, 4)


@pytest.mark.parametrize("splits", [1, 2, 8, 64, 130])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 129, 1025])
def test_splits_and_lengths(dev, length, splits):
    announce(f"fp8 rows length={length} splits={splits}")
    _case(dev, length, 1, 2, 1, 4, 1, 128, torch.bfloat16, 0, length, length, 16, splits)
    _case(dev, length, 1, 2, 0, 4, 1, 128, torch.float16, 0, length, length, 16, splits)


def test_a_context_of_nothing(dev):
    """Extend rows of a request without a context see themselves; a step's rows their ancestors alone."""
    announce("fp8 rows: no context")
    _case(dev, 3, 2, 3, 0, 4, 2, 64, torch.bfloat16, 0, 0, 0, 16, 2)
    _case(dev, 4, 2, 3, 2, 4, 2, 64, torch.bfloat16, 0, 0, 0, 16, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spread", [4.0, 12.0])
def test_scales_far_apart(dev, dtype, spread):
    """Pages whose sizes differ by powers of ten: a weight times a scale would leave fp16's range."""
    announce(f"fp8 rows: scales spread {spread} {dtype}")
    gen = torch.Generator().manual_seed(int(spread))
    page, pages, hkv, dim = 16, 12, 2, 64
    keys, ks = _cache(gen, pages, page, hkv, dim, 0.2)
    values, vs = _cache(gen, pages, page, hkv, dim, 0.2)
    vs = vs * torch.exp(-spread * torch.rand(pages, hkv, generator=gen))  # (the output stays in fp16's range)
    vs[5], vs[7, 0] = 0.0, 0.0
    table = torch.randperm(pages, generator=gen).view(1, -1).int()
    seq = torch.tensor([150])
    q = torch.randn(4, 8, dim, generator=gen).to(dtype)
    args = [t.to(dev) for t in (q, keys, values, ks, vs, table, seq)]
    got = _launch(dev, *args, None, rows=4, step=0, window=0, splits=2, table_page=page)
    _compare(got, q, _wide(keys, ks), _wide(values, vs), table, seq, None, rows_per_request=4, step=0, window=0, table_page=page)


def test_strides_of_caches_and_scales(dev):
    """K and V as halves of one [blocks, heads, page, 2 D] cache, scales one number a layer, q a part of a wider row."""
    announce("fp8 rows: strided")
    gen = torch.Generator().manual_seed(9)
    page, pages, hkv, dim, bs, rows = 16, 9, 2, 128, 2, 3
    both = torch.randn(pages, hkv, page, 2 * dim, generator=gen).to(torch.float8_e4m3fn)
    table = torch.randperm(pages, generator=gen)[:8].view(2, 4).int()
    seq = torch.tensor([50, 41], dtype=torch.int32)
    wide = torch.randn(bs * rows, 4 + 8, dim, generator=gen).to(torch.bfloat16)
    ks, vs = torch.tensor([[0.02]]), torch.tensor([[0.5]])
    view = lambda t: (t.transpose(1, 2)[..., :dim], t.transpose(1, 2)[..., dim:])  # noqa: E731
    k, v = view(both.to(dev))
    out = torch.full((bs * rows, 11, dim), 3.0, dtype=torch.bfloat16, device=dev)
    _launch(dev, wide.to(dev)[:, 4:8], k, v, ks.to(dev).expand(pages, hkv), vs.to(dev).expand(pages, hkv), table.to(dev), seq.to(dev), None,
            rows=rows, step=0, window=0, splits=2, table_page=page, out=out[:, 5:9])
    k, v = view(both.float().double())
    _compare(out[:, 5:9], wide[:, 4:8], k * float(ks), v * float(vs), table, seq, None, rows_per_request=rows, step=0, window=0,
             table_page=page)
    assert (out[:, :5] == 3).all() and (out[:, 9:] == 3).all()


@pytest.mark.parametrize("step", [0, 2])
def test_nan_behind_a_rows_keys_is_not_seen(dev, step):
    """NaN codes (what pages may hold where nothing was written) behind the last extend rows that count, and in ancestors of
    other rows: rows that do not see them are untouched, rows that do are NaN there."""
    announce(f"fp8 rows: NaN codes step={step}")
    gen = torch.Generator().manual_seed(2)
    page, hkv, dim, rows, hq = 16, 1, 64, 4, 2
    keys, ks = _cache(gen, 6, page, hkv, dim, 0.2)
    values, vs = _cache(gen, 6, page, hkv, dim, 0.2)
    table, seq = torch.arange(6).view(1, 6).int(), torch.tensor([40])
    raw_k, raw_v = keys.view(torch.uint8), values.view(torch.uint8)
    anc = None
    if step:
        anc = torch.tensor([[[40, 44], [41, 45], [42, 46], [43, 47]]], dtype=torch.int32)
        bad = 46  # seen by row 2 alone
    else:
        bad = 42  # the position of row 2: seen by rows 2 and 3
    clean = dict(rows_per_request=rows, step=step, window=0, table_page=page)
    q = torch.randn(rows, hq, dim, generator=gen).to(torch.bfloat16)
    run = lambda: _launch(dev, q.to(dev), keys.to(dev), values.to(dev), ks.to(dev), vs.to(dev), table.to(dev), seq.to(dev),  # noqa: E731
                          None if anc is None else anc.to(dev), rows=rows, step=step, window=0, splits=2, table_page=page)
    base = run().cpu()
    _compare(base, q, _wide(keys, ks), _wide(values, vs), table, seq, anc, **clean)
    raw_v[bad // page, bad % page, 0, 7] = 0x7F
    raw_v[bad // page, bad % page, 0, 63] = 0xFF
    got = run().cpu()
    sees = [False, False, True, not step]
    for r in range(rows):
        want = base[r].clone()
        if sees[r]:
            want[:, [7, 63]] = torch.nan
        assert torch.equal(torch.isnan(got[r]), torch.isnan(want))
        assert torch.equal(got[r][~torch.isnan(want)], want[~torch.isnan(want)])
    raw_v[bad // page, bad % page] = 0
    raw_k[bad // page, bad % page] = 0x7F
    got = run().cpu()
    for r in range(rows):
        assert bool(torch.isnan(got[r]).all()) == sees[r] and bool(torch.isnan(got[r]).any()) == sees[r]


def test_written_pages_read_back_by_a_draft_step(dev):
    """write_kv_pages fills the pages that the step reads, its drafted rows among them."""
    from eagle_harness.vllm.kv_pages import write_kv_pages

    announce("fp8 rows: after write_kv_pages")
    gen = torch.Generator().manual_seed(12)
    bs, rows, step, hq, hkv, dim, page = 2, 2, 2, 8, 2, 128, 16
    lens = torch.tensor([37, 90], dtype=torch.int32)
    table = torch.randperm(16, generator=gen).view(2, 8).int().to(dev)
    keys = torch.zeros(16, page, hkv, dim, dtype=torch.float8_e4m3fn, device=dev)
    values, ks, vs = torch.zeros_like(keys), torch.zeros(16, hkv, device=dev), torch.zeros(16, hkv, device=dev)
    kv = lambda n: torch.randn(n, hkv, dim, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    i32 = dict(dtype=torch.int32, device=dev)
    write_kv_pages(kv(127), kv(127), keys, values, ks, vs, table, torch.zeros(2, **i32), torch.tensor([0, 37, 127], **i32), max_query_len=90)
    write_kv_pages(kv(8), kv(8), keys, values, ks, vs, table, lens.to(dev), torch.tensor([0, 4, 8], **i32), max_query_len=4)
    at = lens[:, None, None] + torch.tensor([[[0, 2], [1, 3]]])
    anc = (table.cpu()[torch.arange(2)[:, None, None], at // page] * page + at % page).int()
    q = torch.randn(bs * rows, hq, dim, generator=gen).to(torch.bfloat16)
    got = _launch(dev, q.to(dev), keys, values, ks, vs, table, lens.to(dev), anc.to(dev), rows=rows, step=step, window=0, splits=4,
                  table_page=page)
    _compare(got, q, _wide(keys.cpu(), ks.cpu()), _wide(values.cpu(), vs.cpu()), table.cpu(), lens, anc, rows_per_request=rows, step=step,
             window=0, table_page=page)


def test_pages_outside_the_cache_are_not_read(dev):
    """Table entries and ancestors that name no page: the call ends, and rows that do not see them are right."""
    announce("fp8 rows: entries outside")
    gen = torch.Generator().manual_seed(1)
    keys, ks = _cache(gen, 4, 16, 1, 64, 0.2)
    values, vs = _cache(gen, 4, 16, 1, 64, 0.2)
    table = torch.tensor([[0, 1, 2, 3], [0, 1 << 30, -1, 4]], dtype=torch.int32)
    seq = torch.tensor([60, 60])
    q = torch.randn(2, 2, 64, generator=gen).to(torch.bfloat16)
    anc = torch.tensor([[[61]], [[-7]]], dtype=torch.int32)
    got = _launch(dev, *[t.to(dev) for t in (q, keys, values, ks, vs, table, seq, anc)], rows=1, step=1, window=0, splits=2, table_page=16)
    _compare(got[:1], q[:1], _wide(keys, ks), _wide(values, vs), table[:1], seq[:1], anc[:1], rows_per_request=1, step=1, window=0,
             table_page=16)


def test_captured_and_replayed(dev):
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention

    announce("fp8 rows captured")
    gen = torch.Generator().manual_seed(3)
    bs, rows, hq, hkv, dim, page = 3, 4, 8, 2, 128, 16
    keys, ks = (t.to(dev) for t in _cache(gen, 64, page, hkv, dim))
    values, vs = (t.to(dev) for t in _cache(gen, 64, page, hkv, dim))
    table = torch.randperm(64, generator=gen)[:60].view(3, 20).int().to(dev)
    seq = torch.tensor([200, 1, 77], dtype=torch.int32, device=dev)
    q = torch.randn(bs * rows, hq, dim, generator=gen).to(torch.bfloat16).to(dev)
    part, lse = torch.empty(bs * hq * 9 * 16, dim, device=dev), torch.empty(bs * hq * 9 * 16, device=dev)

    def call(out):
        rows_attention(q, keys, values, out, part, lse, table, seq, None, rows_per_request=rows, step=0, window=0, scale=dim**-0.5,
                       launch=RowsLaunch(splits=8, block_n=32), table_page=page, k_scale=ks, v_scale=vs)

    out = torch.empty_like(q)
    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for lens in ([300, 16, 5], [15, 280, 200], [0, 31, 32]):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        q.normal_()
        graph.replay()
        got = out.clone()
        again = torch.empty_like(q)
        call(again)
        torch.cuda.synchronize()
        assert torch.equal(got, again)
        _compare(got, q.cpu(), _wide(keys.cpu(), ks.cpu()), _wide(values.cpu(), vs.cpu()), table.cpu(), seq.cpu(), None,
                 rows_per_request=rows, step=0, window=0, table_page=page)
