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
