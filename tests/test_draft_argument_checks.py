"""More of what the sampled draft step's operators take and refuse on the host, beside ``test_draft_refusals.py``; a call that passes
every check is refused by the launch, for its tensors are the host's."""

import pytest
import torch

import test_draft_refusals as known

BF16, I32 = torch.bfloat16, torch.int32


def no_requests(**over):
    return {**dict(q=known.zeros(0, 4, 64, dtype=BF16), table=known.zeros(0, 3), seq=known.zeros(0)), **over}


@pytest.mark.parametrize("over,error", [
    (no_requests(), RuntimeError),
    (no_requests(table=known.zeros(0, 0)), RuntimeError),
    (no_requests(table=known.zeros(0)), ValueError),
    (dict(q=known.zeros(3, 4, 64, dtype=BF16)), ValueError),  # one request of two rows, and a row
    (dict(q=known.zeros(1, 4, 64, dtype=BF16)), ValueError),
    (dict(seq=torch.zeros((), dtype=I32)), ValueError),
])
def test_rows_over_fp8_pages(over, error):
    with pytest.raises(error):
        known.rows(**over)


@pytest.mark.parametrize("count", [0, -2])
def test_rows_a_request(count):
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention

    q, cache = known.zeros(2, 4, 64, dtype=BF16), known.zeros(5, 16, 2, 64, dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        rows_attention(q, cache, cache, torch.zeros_like(q), torch.zeros(192, 64), torch.zeros(192), known.zeros(1, 3), known.zeros(1), None,
                       rows_per_request=count, step=0, window=0, scale=1.0, launch=RowsLaunch(splits=2, block_n=32), table_page=16,
                       k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2))


@pytest.mark.parametrize("name", ["q", "out", "keys", "values"])
@pytest.mark.parametrize("scales", [False, True])
def test_the_tensor_without_a_unit_stride_is_named(name, scales):
    from eagle_harness.kernels._native import NotCovered
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention

    cached = torch.float8_e4m3fn if scales else BF16
    x = dict(q=known.zeros(2, 4, 64, dtype=BF16), out=known.zeros(2, 4, 64, dtype=BF16), keys=known.zeros(5, 16, 2, 64, dtype=cached),
             values=known.zeros(5, 16, 2, 64, dtype=cached))
    x[name] = torch.zeros(*x[name].shape[:-1], 128, dtype=x[name].dtype)[..., ::2]
    ks, vs = (torch.ones(5, 2), torch.ones(5, 2)) if scales else (None, None)
    with pytest.raises(NotCovered, match=f"^{name} must"):
        rows_attention(x["q"], x["keys"], x["values"], x["out"], torch.zeros(192, 64), torch.zeros(192), known.zeros(1, 3), known.zeros(1), None,
                       rows_per_request=2, step=0, window=0, scale=1.0, launch=RowsLaunch(splits=2, block_n=32), table_page=16,
                       k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("seed", range(40))
def test_tensors_known_to_be_apart(seed):
    """Against the bytes themselves: what is called apart shares none; and layouts that are used are called apart."""
    import random

    from eagle_harness.kernels._native import apart

    rng = random.Random(seed)

    def touched(at, dims, width):
        places = [at]
        for count, stride in dims:
            places = [p + i * stride for p in places for i in range(count)]
        return {p + i for p in places for i in range(width)}

    for _ in range(400):
        steps = rng.choice(([24, 96], [96, 24], [8, 40], [0, 16], [16, 16], [30, 7]))
        other = steps if rng.random() < 0.7 else [rng.randint(0, 100) for _ in steps]
        one = (rng.randint(0, 60), tuple((rng.randint(0, 4), s) for s in steps), rng.randint(1, 30))
        two = (rng.randint(0, 60), tuple((rng.randint(0, 4), s) for s in other), rng.randint(1, 30))
        if touched(*one) & touched(*two):
            assert not apart(*one, *two)
    assert apart(1000, ((5, 80),), 40, 1040, ((5, 80),), 40) and not apart(1000, ((5, 80),), 40, 1038, ((5, 80),), 40)
    assert apart(0, ((3, 96), (2, 48)), 24, 24, ((3, 96), (2, 48)), 24)  # halves of every head
    assert apart(0, ((3, 96), (2, 12)), 12, 24, ((3, 96), (2, 12)), 12)  # heads of one packed row
    assert apart(0, ((1, 7), (4, 16)), 8, 8, ((4, 16),), 8)


@pytest.mark.parametrize("at,error", [(10, RuntimeError), (9, ValueError), (5, ValueError), (0, ValueError)])
def test_outputs_in_other_columns_of_the_logits_store(at, error):
    """Rows of one wider buffer: columns of their own are taken (and refused by the launch alone), shared ones are not."""
    wide = torch.zeros(3, 20)
    with pytest.raises(error):
        known.draw(logits=wide[:, :10], probs=wide[:, at : at + 10])
    if at:
        with pytest.raises(error):
            known.draw(truncate=True, logits=wide[:, :10], out=wide[:, at : at + 10])
        with pytest.raises(error):
            known.draw(truncate=True, logits=wide[:, at : at + 10], out=wide[:, :10])


def heads_of(first, last, lead=0, tokens=4, heads=5, dim=16):
    return lambda store: store[lead:].view(-1)[: tokens * heads * dim].view(tokens, heads, dim)[:, first:last]


@pytest.mark.parametrize("q,out,error", [
    (heads_of(0, 2), heads_of(2, 4), RuntimeError),  # other heads of one packed row
    (heads_of(3, 5), heads_of(0, 2), RuntimeError),
    (heads_of(0, 2), heads_of(1, 3), ValueError),
    (heads_of(0, 2), heads_of(2, 4, lead=8), RuntimeError),
    (heads_of(0, 2), heads_of(1, 3, lead=8), ValueError),
    (lambda s: s[:320].view(4, 5, 16)[..., :8], lambda s: s[:320].view(4, 5, 16)[..., 8:], RuntimeError),  # halves of every head
    (lambda s: s[:320].view(5, 4, 16).transpose(0, 1)[:, :2], lambda s: s[:320].view(5, 4, 16).transpose(0, 1)[:, 2:4], RuntimeError),
    (lambda s: s[:320].view(5, 4, 16).transpose(0, 1)[:, :2], lambda s: s[:320].view(5, 4, 16).transpose(0, 1)[:, 1:3], ValueError),
])
def test_rotated_rows_beside_their_inputs(q, out, error):
    store = torch.zeros(400)
    with pytest.raises(error):
        known.rotate(q=q(store), q_out=out(store), k=None)


@pytest.mark.parametrize("at,error", [(4, RuntimeError), (5, RuntimeError), (3, ValueError), (0, ValueError)])
def test_a_batch_table_beside_the_block_table(at, error):
    wide = known.zeros(3, 9)
    with pytest.raises(error):
        known.maps(table=wide[:, :4], batch=wide[:2, at : at + 4])


@pytest.mark.parametrize("page", [(1 << 31), (1 << 32) + 16, -16])
def test_page_sizes_past_32_bits(page):
    for call in (known.resize, known.maps):
        with pytest.raises(ValueError):
            call(page=page)


@pytest.mark.parametrize("scales", [False, True])
def test_windows_and_table_pages_past_32_bits(monkeypatch, scales):
    """A window longer than 32 bits is the longest, not what its low bits say; a table page is refused."""
    from eagle_harness.kernels import _native, row_attention

    given = []
    monkeypatch.setattr(_native, "launch", lambda name, args, device: given.append(args.rows if scales else args))
    q, cache = known.zeros(2, 4, 64, dtype=BF16), known.zeros(5, 16, 2, 64, dtype=torch.float8_e4m3fn if scales else BF16)
    ks, vs = (torch.ones(5, 2), torch.ones(5, 2)) if scales else (None, None)

    def call(window, page=16):
        row_attention.rows_attention(q, cache, cache, torch.zeros_like(q), torch.zeros(192, 64), torch.zeros(192), known.zeros(1, 3),
                                     known.zeros(1), None, rows_per_request=2, step=0, window=window, scale=1.0,
                                     launch=row_attention.RowsLaunch(splits=2, block_n=32), table_page=page, k_scale=ks, v_scale=vs)

    for window, want in ((0, 0), (5, 5), ((1 << 31) - 1, (1 << 31) - 1), (1 << 31, (1 << 31) - 1), ((1 << 32) + 5, (1 << 31) - 1)):
        call(window)
        assert given[-1].window == want
    for page in (1 << 31, (1 << 32) + 16, -(1 << 32) + 16):
        with pytest.raises(ValueError):
            call(0, page)
