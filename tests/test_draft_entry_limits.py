"""More of what the C entries of the sampled draft step's operators check before any launch, beside ``test_draft_entry_checks.py``; its
calls and its pointers, so only where there is no GPU."""

import pytest
import torch

from eagle_harness.kernels import _native
from test_draft_entry_checks import NOT_COVERED, OK, ON, fp8_rows, rotary, sampled

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that pass the checks would be launched")


def test_copies_of_padded_rows_are_truncated_rows():
    call = _native.library().eagle4_sample_rows
    cut = dict(coins=0, tokens=0, draws=0, out=ON, stride_out=9, out_kind=2, copy_padded=1)
    assert call(sampled(**cut), None) not in (OK, NOT_COVERED)
    assert call(sampled(out=ON, stride_out=9, out_kind=1, copy_padded=1), None) == NOT_COVERED
    assert call(sampled(copy_padded=1), None) == NOT_COVERED


def test_rotary_tokens_past_a_launch():
    """2^24 workgroups of 256 threads are more than a launch takes; these shapes have 64 tokens a workgroup, and wide heads one."""
    call = _native.library().eagle4_rotary
    assert call(rotary(tokens=1 << 30), None) == NOT_COVERED
    assert call(rotary(tokens=(1 << 30) - 64), None) not in (OK, NOT_COVERED)
    wide = dict(dim=1024, half=512, q_heads=64, stride_qh=1024, stride_kh=1024, stride_qoh=1024, stride_koh=1024)
    assert call(rotary(tokens=1 << 24, **wide), None) == NOT_COVERED
    assert call(rotary(tokens=(1 << 24) - 1, **wide), None) not in (OK, NOT_COVERED)


def test_rows_over_fp8_pages_past_the_merges_launch():
    """2^26 pairs of a row and a head of 256, four a workgroup of the merge: refused before the first launch."""
    call = _native.library().eagle4_row_attention_fp8
    many = dict(step=0, ancestors=0, head_dim=256, heads=16, kv_heads=1, rows_per_request=64, rows_padded=64, splits=1, part_rows=1 << 40,
                stride_q_row=4096, stride_q_head=256, stride_o_row=4096, stride_o_head=256)
    scales = dict(table_width=4, table_height=65535)
    assert call(fp8_rows(scales, bs=65535, **many), None) not in (OK, NOT_COVERED)
    assert call(fp8_rows(scales, bs=65535, **{**many, "heads": 17}), None) == NOT_COVERED
