"""What the sampled draft step's operators refuse, before any launch and on the CPU: arguments that do not fit raise ValueError,
layouts and types that the kernels do not address raise NotCovered, host tensors that pass are refused by the launch. And the
frequencies of rotary positions, which are made on the host."""

import math

import pytest
import torch

from eagle_harness.kernels._native import NotCovered

I32, F64 = torch.int32, torch.float64


def draw(truncate=False, **over):
    from eagle_harness.vllm.sampling import draw_tokens, truncate_logits

    x = dict(logits=torch.zeros(3, 10), coins=torch.zeros(3, 2), t=torch.ones(3), k=torch.zeros(3, dtype=I32), p=torch.ones(3),
             m=torch.zeros(3), entries=None, probs=None, out=None)
    x.update(over)
    if truncate:
        return truncate_logits(x["logits"], x["t"], x["k"], x["p"], x["m"], entries=x["entries"], out=x["out"])
    return draw_tokens(x["logits"], x["coins"], x["t"], x["k"], x["p"], x["m"], entries=x["entries"], probs=x["probs"])


SHARED = [
    (dict(logits=torch.zeros(30)), ValueError),
    (dict(logits=torch.zeros(10, 3).t()), NotCovered),
    (dict(logits=torch.zeros(3, 10, dtype=F64)), NotCovered),
    (dict(logits=torch.zeros(3, 0)), NotCovered),
    (dict(logits=torch.zeros(3, (1 << 18) + 1, dtype=torch.bfloat16)), NotCovered),
    (dict(t=torch.ones(2)), ValueError),
    (dict(t=torch.ones(3, dtype=F64)), ValueError),
    (dict(t=torch.ones(3, 1)), ValueError),
    (dict(k=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(k=torch.zeros(2, dtype=I32)), ValueError),
    (dict(p=torch.ones(6)[::2]), ValueError),
    (dict(m=torch.zeros(4)), ValueError),
    (dict(entries=torch.zeros(2, dtype=I32)), ValueError),
    (dict(entries=torch.zeros(3)), NotCovered),
    (dict(entries=torch.zeros(3, dtype=I32), t=torch.ones(0), k=None, p=None, m=None), ValueError),
    (dict(), RuntimeError),  # host tensors
    (dict(k=None, p=None, m=None), RuntimeError),
]


@pytest.mark.parametrize("over,error", SHARED + [
    (dict(coins=torch.zeros(2, 2)), ValueError),
    (dict(coins=torch.zeros(3, 65)), ValueError),
    (dict(coins=torch.zeros(3, 0)), ValueError),
    (dict(coins=torch.zeros(())), ValueError),
    (dict(coins=torch.zeros(3, 2, dtype=F64)), ValueError),
    (dict(coins=torch.zeros(3, 4)[:, ::2]), ValueError),
    (dict(probs=torch.zeros(3, 9)), ValueError),
    (dict(probs=torch.zeros(3, 10, dtype=F64)), NotCovered),
    (dict(probs=torch.zeros(10, 3).t()), NotCovered),
    (dict(probs=torch.zeros(1, 10).expand(3, 10)), NotCovered),
    (dict(probs=torch.zeros(3, 10, dtype=torch.float16)), RuntimeError),
    (dict(zip(("logits", "probs"), [torch.zeros(3, 10)] * 2)), ValueError),
])
def test_draw_tokens(over, error):
    with pytest.raises(error):
        draw(**over)


def overlapping():
    store = torch.zeros(40)
    return dict(logits=store[:30].view(3, 10), out=store[1:31].view(3, 10))


@pytest.mark.parametrize("over,error", SHARED + [
    (dict(out=torch.zeros(3, 9)), ValueError),
    (dict(out=torch.zeros(3, 10, dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros(1, 10).expand(3, 10)), NotCovered),
    (overlapping(), ValueError),
])
def test_truncate_logits(over, error):
    with pytest.raises(error):
        draw(truncate=True, **over)


def rotate(**over):
    from eagle_harness.vllm.rotary import rotate_rows

    x = dict(q=torch.zeros(4, 2, 16), k=torch.zeros(4, 1, 16), positions=torch.zeros(4, dtype=I32), f=torch.ones(4, dtype=F64),
             q_out=None, k_out=None)
    x.update(over)
    return rotate_rows(x["q"], x["k"], x["positions"], x["f"], q_out=x["q_out"], k_out=x["k_out"])


def shifted():
    store = torch.zeros(4 * 2 * 16 + 8)
    return dict(q=store[:128].view(4, 2, 16), q_out=store[8:136].view(4, 2, 16), k=None)


@pytest.mark.parametrize("over,error", [
    (dict(q=torch.zeros(4, 32)), ValueError),
    (dict(q=torch.zeros(4, 2, 16, dtype=F64)), NotCovered),
    (dict(q=torch.zeros(4, 16, 2).transpose(1, 2)), NotCovered),
    (dict(k=torch.zeros(3, 1, 16)), ValueError),
    (dict(k=torch.zeros(4, 1, 8)), ValueError),
    (dict(k=torch.zeros(4, 1, 16, dtype=torch.bfloat16)), ValueError),
    (dict(f=torch.ones(4)), ValueError),
    (dict(f=torch.ones(9, dtype=F64)), ValueError),
    (dict(f=torch.ones(0, dtype=F64)), ValueError),
    (dict(f=torch.ones(8, dtype=F64)[::2]), ValueError),
    (dict(positions=torch.zeros(3, dtype=I32)), ValueError),
    (dict(positions=torch.zeros(4)), NotCovered),
    (dict(positions=torch.zeros(1, 4, dtype=I32)), ValueError),
    (dict(q_out=torch.zeros(4, 2, 16)), ValueError),  # for q alone
    (dict(q_out=torch.zeros(4, 1, 16), k_out=torch.zeros(4, 1, 16)), ValueError),
    (dict(k=None, k_out=torch.zeros(4, 1, 16)), ValueError),
    (dict(q=torch.zeros(1, 2, 16).expand(4, 2, 16), k=None), ValueError),
    (dict(q_out=torch.zeros(4, 1, 16).expand(4, 2, 16), k=None), ValueError),
    (shifted(), ValueError),
    (dict(q=torch.zeros(200).as_strided((4, 2, 16), (16, 8, 1)), k=None), ValueError),  # heads that overlap
    (dict(q=torch.zeros(200).as_strided((4, 2, 16), (24, 16, 1)), k=None), ValueError),  # tokens that do
    (dict(q=torch.zeros(200).as_strided((4, 2, 16), (16, 56, 1)), k=None), ValueError),
    (dict(q=torch.zeros(200).as_strided((4, 2, 16), (16, 64, 1)), k=None), RuntimeError),  # heads before tokens: none
    (dict(), RuntimeError),
    (dict(k=None), RuntimeError),
])
def test_rotate_rows(over, error):
    with pytest.raises(error):
        rotate(**over)


def test_frequencies():
    from eagle_harness.vllm.rotary import rotary_frequencies

    f, factor = rotary_frequencies(8, 10000.0)
    assert f.dtype == F64 and factor == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=F64), rtol=1e-12)
    g, factor = rotary_frequencies(8, scaling="linear", stretch=4.0)
    assert torch.allclose(g, f / 4, rtol=1e-12) and factor == 1.0
    g, _ = rotary_frequencies(8, scaling="ntk", stretch=4.0)
    assert float(g[0]) == 1.0 and math.isclose(float(g[3]), float(f[3]) / 4, rel_tol=1e-12)
    f, _ = rotary_frequencies(128)
    g, factor = rotary_frequencies(128, scaling="yarn", stretch=8.0, trained=4096)
    ratio = f / g
    assert float(ratio[0]) == 1.0 and math.isclose(float(ratio[-1]), 8.0, rel_tol=1e-12)
    assert bool((ratio[1:] >= ratio[:-1] - 1e-12).all()) and math.isclose(factor, 0.1 * math.log(8.0) + 1)
    # a pair that turns more than 32 times in 4096 positions stays, one that turns less than once is stretched whole
    turns = f * 4096 / (2 * math.pi)
    assert bool((ratio[turns > 40] == 1).all()) and torch.allclose(ratio[turns < 0.8], torch.tensor(8.0, dtype=F64), rtol=1e-12)
    assert torch.equal(rotary_frequencies(128, scaling="yarn", stretch=1.0, trained=4096)[0], f)


@pytest.mark.parametrize("args", [dict(dim=7), dict(dim=0), dict(dim=8, base=1.0), dict(dim=8, stretch=0.5), dict(dim=8, scaling="other"),
                                  dict(dim=2, scaling="ntk"), dict(dim=8, scaling="yarn"), dict(dim=8, scaling="yarn", trained=64, fast=1.0)])
def test_frequencies_refuse(args):
    from eagle_harness.vllm.rotary import rotary_frequencies

    with pytest.raises(ValueError):
        rotary_frequencies(args.pop("dim"), **args)


def zeros(*n, dtype=I32):
    return torch.zeros(*n, dtype=dtype)


def resize(**over):
    from eagle_harness.vllm.page_tables import resize_tables

    x = dict(table=zeros(3, 4), pages=zeros(3), idx=zeros(2), lens=zeros(2), free=zeros(9), n=zeros(1), page=16)
    x.update(over)
    return resize_tables(x["table"], x["pages"], x["idx"], x["lens"], x["free"], x["n"], x["page"])


TABLES = [
    (dict(table=zeros(12)), ValueError),
    (dict(table=zeros(3, 4, dtype=torch.int64)), ValueError),
    (dict(table=zeros(0, 4)), ValueError),
    (dict(table=zeros(4, 3).t()), NotCovered),
    (dict(table=zeros(1, 4).expand(3, 4)), NotCovered),
    (dict(pages=zeros(2)), ValueError),
    (dict(pages=zeros(3, dtype=torch.int64)), ValueError),
    (dict(pages=zeros(6)[::2]), ValueError),
    (dict(idx=zeros(2, 1)), ValueError),
    (dict(idx=torch.zeros(2)), NotCovered),
    (dict(page=0), ValueError),
    (dict(), RuntimeError),
]


@pytest.mark.parametrize("over,error", TABLES + [
    (dict(lens=zeros(1)), ValueError),
    (dict(lens=torch.zeros(2)), NotCovered),
    (dict(free=zeros(9, dtype=torch.int64)), ValueError),
    (dict(free=zeros(18)[::2]), ValueError),
    (dict(n=zeros(2)), ValueError),
    (dict(n=zeros(1, dtype=torch.int64)), ValueError),
])
def test_resize_tables(over, error):
    with pytest.raises(error):
        resize(**over)


def maps(**over):
    from eagle_harness.vllm.page_tables import slot_maps

    x = dict(table=zeros(3, 4), pages=zeros(3), idx=zeros(2), context=zeros(2), starts=zeros(3), page=16, slots=zeros(9, dtype=torch.int64),
             batch=zeros(2, 4))
    x.update(over)
    return slot_maps(x["table"], x["pages"], x["idx"], x["context"], x["starts"], x["page"], slots=x["slots"], batch_table=x["batch"])


@pytest.mark.parametrize("over,error", TABLES + [
    (dict(context=zeros(1)), ValueError),
    (dict(starts=zeros(2)), ValueError),
    (dict(slots=zeros(9)), ValueError),
    (dict(slots=zeros(18, dtype=torch.int64)[::2]), ValueError),
    (dict(batch=zeros(1, 4)), ValueError),
    (dict(batch=zeros(2, 5)), ValueError),
    (dict(batch=zeros(1, 4).expand(2, 4)), NotCovered),
    (dict(zip(("table", "batch"), [zeros(3, 4)] * 2)), ValueError),
    (dict(context=zeros(2, 2)), ValueError),
    (dict(starts=zeros(3, 2)), ValueError),
    (dict(batch=None), RuntimeError),
])
def test_slot_maps(over, error):
    with pytest.raises(error):
        maps(**over)


def rows(**over):
    from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention

    fp8 = torch.float8_e4m3fn
    x = dict(q=zeros(2, 4, 64, dtype=torch.bfloat16), keys=zeros(5, 16, 2, 64, dtype=fp8), values=zeros(5, 16, 2, 64, dtype=fp8),
             ks=torch.ones(5, 2), vs=torch.ones(5, 2), table=zeros(1, 3), out=None, seq=zeros(1), step=0, anc=None)
    x.update(over)
    out = torch.zeros_like(x["q"]) if x["out"] is None else x["out"]
    part = x.get("part", torch.zeros(4 * 3 * 16, 64))
    return rows_attention(x["q"], x["keys"], x["values"], out, part, x.get("lse", torch.zeros(4 * 3 * 16)), x["table"],
                          x["seq"], x["anc"], rows_per_request=2, step=x["step"], window=0, scale=1.0, launch=RowsLaunch(splits=2, block_n=32),
                          table_page=16, k_scale=x["ks"], v_scale=x["vs"])


@pytest.mark.parametrize("over,error", [
    (dict(ks=None), ValueError),
    (dict(vs=None), ValueError),
    (dict(ks=torch.ones(4, 2)), ValueError),
    (dict(vs=torch.ones(5, 1)), ValueError),
    (dict(vs=torch.ones(10)), ValueError),
    (dict(ks=torch.ones(5, 2, dtype=F64)), ValueError),
    (dict(values=None), NotCovered),
    (dict(keys=zeros(5, 16, 2, 64, dtype=torch.bfloat16)), NotCovered),
    (dict(values=zeros(4, 16, 2, 64, dtype=torch.float8_e4m3fn)), ValueError),
    (dict(q=zeros(2, 4, 64, dtype=torch.float32)), NotCovered),
    (dict(out=zeros(2, 4, 64, dtype=torch.float16)), NotCovered),
    (dict(table=zeros(1, 0)), ValueError),
    (dict(table=zeros(3)), ValueError),
    (dict(out=zeros(2, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(keys=zeros(5, 16, 2, 128, dtype=torch.float8_e4m3fn), values=zeros(5, 16, 2, 128, dtype=torch.float8_e4m3fn)), ValueError),
    (dict(seq=zeros(0)), ValueError),
    (dict(step=2, anc=zeros(1, 2, 1)), ValueError),
    (dict(step=2, anc=zeros(1, 1, 2)), ValueError),
    (dict(step=2, anc=None), ValueError),
    (dict(step=2, anc=zeros(1, 2, 2)), RuntimeError),
    (dict(keys=zeros(0, 16, 2, 64, dtype=torch.float8_e4m3fn), values=zeros(0, 16, 2, 64, dtype=torch.float8_e4m3fn)), ValueError),
    (dict(q=zeros(4, 4, 64, dtype=torch.bfloat16), seq=zeros(2)), ValueError),  # two requests, one row of the table
    (dict(part=torch.zeros(4 * 3 * 16, 32)), ValueError),
    (dict(part=torch.zeros(4 * 3 * 16 * 64)), ValueError),
    (dict(lse=torch.zeros(2 * 4 * 3 * 16)[::2]), ValueError),
    (dict(ks=None, vs=None), NotCovered),  # fp8 caches without scales
    (dict(), RuntimeError),
])
def test_rows_attention_over_fp8_pages(over, error):
    with pytest.raises(error):
        rows(**over)
