"""The C entries' own checks of the sampled draft step's operators (status -1 before any launch), for callers that bind them directly:
each case differs in one argument from a call that passes every check and comes to a launch. The pointers are none, so this
runs only where there is no GPU: the launch itself then fails, with the runtime's status."""

import pytest
import torch

from eagle_harness.kernels import _native

I32 = torch.int32
ON = 1 << 20  # a pointer that is never followed
OK, NOT_COVERED = 0, -1
TAB = _native.itab(torch.zeros(4, 4, dtype=I32))
NO_TAB = _native.itab(None)

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that pass the checks would be launched")


def sampled(**over):
    return _native.SampleRowsArgs(**{**dict(
        logits=ON, stride_row=9, entries=TAB, temperature=ON, coins=ON, tokens=ON, rows=4, num_entries=2, vocab=9, draws=2), **over})


def rotary(**over):
    return _native.RotaryArgs(**{**dict(
        q=ON, k=ON, q_out=ON + 4096, k_out=ON + 4096, stride_qt=64, stride_qh=16, stride_kt=64, stride_kh=16, stride_qot=64, stride_qoh=16,
        stride_kot=64, stride_koh=16, positions=TAB, frequencies=ON, factor=1.0, tokens=3, q_heads=2, k_heads=1, dim=16, half=4), **over})


def tables(**over):
    return _native.ResizeTablesArgs(**{**dict(
        block_table=ON, stride_table=8, num_pages=ON, idx_mapping=TAB, lens=TAB, free_pages=ON, num_free=ON, capacity=9, num_reqs=2,
        slots=3, max_pages=8, page=16), **over})


def maps(**over):
    return _native.SlotMapsArgs(**{**dict(
        block_table=ON, stride_table=8, num_pages=ON, idx_mapping=TAB, context_lens=TAB, query_start_loc=TAB, slots=ON, batch_table=ON,
        stride_batch=8, rows=9, num_reqs=2, state_slots=3, max_pages=8, page=16), **over})


def fp8_rows(scales=None, **over):
    rows = _native.RowAttnArgs(**{**dict(
        q=ON, stride_q_row=256, stride_q_head=64, keys=ON, values=ON, k_stride_page=1024, k_stride_slot=128, k_stride_head=64,
        v_stride_page=1024, v_stride_slot=128, v_stride_head=64, out=ON, stride_o_row=256, stride_o_head=64, part_out=ON, part_lse=ON,
        part_rows=1 << 20, table=ON, stride_table=4, seq_lens=TAB, ancestors=ON, max_depth=3, table_page=16, cache_page=16, bs=2,
        rows_per_request=2, rows_padded=16, heads=4, kv_heads=2, head_dim=64, dtype=0, step=3, window=0, splits=2, scale=1.0), **over})
    return _native.RowAttnFp8Args(**{**dict(rows=rows, k_scale=ON, v_scale=ON, stride_ksb=2, stride_ksh=1, stride_vsb=2, stride_vsh=1,
                                            table_height=2, table_width=4, num_blocks=5), **(scales or {})})


CALLS = {"eagle4_sample_rows": sampled, "eagle4_rotary": rotary, "eagle4_resize_tables": tables, "eagle4_slot_maps": maps,
         "eagle4_row_attention_fp8": fp8_rows}


@pytest.mark.parametrize("name,over", [
    ("eagle4_sample_rows", {}), ("eagle4_sample_rows", dict(entries=NO_TAB)),
    ("eagle4_sample_rows", dict(out=ON, stride_out=9, out_kind=1, out_dtype=1)),
    ("eagle4_sample_rows", dict(coins=0, tokens=0, draws=0, out=ON, stride_out=9, out_kind=2)),
    ("eagle4_rotary", {}), ("eagle4_rotary", dict(k=0, k_out=0, k_heads=0)), ("eagle4_rotary", dict(q_out=ON, k_out=ON)),
    ("eagle4_resize_tables", {}), ("eagle4_slot_maps", {}), ("eagle4_slot_maps", dict(batch_table=0)),
    ("eagle4_row_attention_fp8", {}), ("eagle4_row_attention_fp8", dict(step=0, ancestors=0)),
])
def test_the_base_comes_to_a_launch(name, over):
    assert getattr(_native.library(), name)(CALLS[name](**over), None) not in (OK, NOT_COVERED)


@pytest.mark.parametrize("name,over", [
    ("eagle4_sample_rows", dict(rows=0, logits=0)), ("eagle4_rotary", dict(tokens=0, q=0)), ("eagle4_rotary", dict(q_heads=0, k_heads=0)),
    ("eagle4_resize_tables", dict(num_reqs=0)), ("eagle4_slot_maps", dict(rows=0, num_reqs=0)), ("eagle4_row_attention_fp8", dict(bs=0)),
])
def test_nothing_to_do(name, over):
    assert getattr(_native.library(), name)(CALLS[name](**over), None) == OK


@pytest.mark.parametrize("over", [
    dict(logits=0), dict(logits=ON + 1), dict(temperature=0), dict(vocab=0), dict(vocab=(1 << 18) + 1), dict(rows=-1), dict(rows=(1 << 20) + 1),
    dict(num_entries=0), dict(dtype=3), dict(draws=65), dict(draws=0), dict(tokens=0), dict(coins=0), dict(stride_row=-1),
    dict(coins=0, tokens=0, draws=0), dict(entries=_native.ITab(ON, 1, 0, 2, 0)), dict(out=ON, stride_out=9, out_kind=0),
    dict(out=ON, stride_out=9, out_kind=3), dict(out=ON, stride_out=8, out_kind=1), dict(out=ON, stride_out=9, out_kind=2, out_dtype=2),
    dict(out=ON + 2, stride_out=9, out_kind=1, out_dtype=2), dict(out=ON, stride_out=9, out_kind=1, out_dtype=5)])
def test_sampled_rows_refuse(over):
    assert _native.library().eagle4_sample_rows(sampled(**over), None) == NOT_COVERED


@pytest.mark.parametrize("over", [
    dict(q=0), dict(q_out=0), dict(k=0), dict(k_out=0), dict(positions=NO_TAB), dict(frequencies=0), dict(half=0), dict(half=9),
    dict(half=513, dim=2048), dict(tokens=-1), dict(q_heads=-1), dict(dtype=3), dict(q_out=ON), dict(k_out=ON), dict(q_heads=4096),
    dict(dim=(1 << 16) + 1)])
def test_rotary_refuses(over):
    assert _native.library().eagle4_rotary(rotary(**over), None) == NOT_COVERED


@pytest.mark.parametrize("over", [
    dict(block_table=0), dict(num_pages=0), dict(idx_mapping=NO_TAB), dict(lens=NO_TAB), dict(free_pages=0), dict(num_free=0),
    dict(capacity=-1), dict(capacity=1 << 31), dict(num_reqs=-1), dict(slots=0), dict(max_pages=0), dict(page=0), dict(stride_table=7)])
def test_resize_tables_refuses(over):
    assert _native.library().eagle4_resize_tables(tables(**over), None) == NOT_COVERED


@pytest.mark.parametrize("over", [
    dict(block_table=0), dict(num_pages=0), dict(idx_mapping=NO_TAB), dict(context_lens=NO_TAB), dict(query_start_loc=NO_TAB), dict(slots=0),
    dict(rows=-1), dict(num_reqs=-1), dict(state_slots=0), dict(max_pages=0), dict(page=0), dict(stride_table=7), dict(stride_batch=7)])
def test_slot_maps_refuses(over):
    assert _native.library().eagle4_slot_maps(maps(**over), None) == NOT_COVERED


@pytest.mark.parametrize("over", [
    dict(q=0), dict(q=ON + 8), dict(keys=0), dict(keys=ON + 8), dict(values=0), dict(out=0), dict(out=ON + 4), dict(part_out=0),
    dict(part_lse=0), dict(table=0), dict(seq_lens=NO_TAB), dict(ancestors=0), dict(max_depth=2), dict(step=-1), dict(splits=0),
    dict(head_dim=96), dict(dtype=2), dict(heads=3), dict(kv_heads=0), dict(rows_padded=1), dict(part_rows=100), dict(table_page=0),
    dict(cache_page=0), dict(k_stride_slot=120), dict(v_stride_head=8), dict(stride_q_row=252), dict(stride_o_head=2), dict(bs=65536)])
def test_rows_over_fp8_pages_refuse(over):
    assert _native.library().eagle4_row_attention_fp8(fp8_rows(**over), None) == NOT_COVERED


@pytest.mark.parametrize("scales", [dict(k_scale=0), dict(v_scale=0), dict(table_height=0), dict(table_width=0), dict(num_blocks=0)])
def test_scales_and_tables_that_rows_over_fp8_pages_refuse(scales):
    assert _native.library().eagle4_row_attention_fp8(fp8_rows(scales), None) == NOT_COVERED
