"""The C entries' own checks (status -1 before any launch), for callers that bind them directly: each case differs in one argument
from a call that passes every check and comes to a launch. The pointers are none, so this runs only where there is no GPU: the
launch itself then fails, with the runtime's status."""

import pytest
import torch

from eagle_harness.kernels import _native

I32 = torch.int32
ON = 1 << 20  # a pointer that is never followed
NOT_COVERED = -1

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that pass the checks would be launched")


def sampled(**over):
    tab = _native.itab(torch.zeros(4, 4, dtype=I32))
    return _native.SampleTreeArgs(**{**dict(
        logits=ON, drafted=tab, cu_num_logits=tab, idx_mapping=tab, parents=tab, coins=ON, final_coins=ON, temperature=ON,
        sampled=ON, num_sampled=ON, path=ON, path_len=ON, workspace=ON, workspace_bytes=1 << 40, rows=4, num_reqs=1, width=4,
        vocab=9, slots=4), **over})


def test_the_sampled_walks_base_comes_to_a_launch():
    lib = _native.library()
    need = lib.eagle4_sample_tree_workspace(sampled())
    assert need > 0
    assert lib.eagle4_sample_tree(sampled(workspace_bytes=need), None) not in (0, NOT_COVERED)
    assert lib.eagle4_sample_tree(sampled(probs=ON, prob_dtype=2), None) not in (0, NOT_COVERED)
    assert lib.eagle4_sample_tree(sampled(workspace_bytes=need - 1), None) == NOT_COVERED


@pytest.mark.parametrize("over", [dict(width=0), dict(width=65), dict(vocab=0), dict(slots=0), dict(num_reqs=65536), dict(rows=-1)])
def test_sizes_that_the_sampled_walk_does_not_cover(over):
    assert _native.library().eagle4_sample_tree_workspace(sampled(**over)) == -1
    assert _native.library().eagle4_sample_tree(sampled(**over), None) == NOT_COVERED


@pytest.mark.parametrize("over", [dict(workspace=0), dict(workspace=ON + 8), dict(logits=0), dict(coins=0), dict(final_coins=0),
                                  dict(temperature=0), dict(sampled=0), dict(num_sampled=0), dict(path=0), dict(path_len=0),
                                  dict(dtype=3), dict(probs=ON, prob_dtype=4), dict(drafted=_native.ITab()),
                                  dict(parents=_native.itab(None)), dict(cu_num_logits=_native.itab(None)),
                                  dict(idx_mapping=_native.itab(None))])
def test_arguments_that_the_sampled_walk_refuses(over):
    assert _native.library().eagle4_sample_tree(sampled(**over), None) == NOT_COVERED


def latent(**over):
    tab = _native.itab(torch.zeros(4, 4, dtype=I32))
    return _native.LatentAttnArgs(**{**dict(
        q=ON, stride_qt=4096, stride_qh=576, latent_new=ON, stride_nt=576, cache=ON, stride_cb=576 * 16, stride_cs=576,
        block_table=tab, context_lens=tab, query_start_loc=tab, masks=ON, stride_mask=1, out=ON, stride_ot=4096, stride_oh=512,
        workspace=ON, workspace_bytes=1 << 40, tokens=1, scale=1.0, num_reqs=1, heads=16, rank=512, rope=64, page=16,
        max_query_len=1, max_blocks=4, num_blocks=4), **over})


def test_latent_attentions_base_comes_to_a_launch():
    lib = _native.library()
    assert lib.eagle4_latent_attention(latent(), None) not in (0, NOT_COVERED)
    assert lib.eagle4_latent_attention(latent(cache_dtype=3, scale_page=ON), None) not in (0, NOT_COVERED)
    assert lib.eagle4_latent_attention(latent(tokens=0, q=0, latent_new=0, out=0), None) not in (0, NOT_COVERED)
    assert lib.eagle4_latent_attention(latent(num_blocks=0, cache=0), None) not in (0, NOT_COVERED)


@pytest.mark.parametrize("over", [dict(q=0), dict(latent_new=0), dict(out=0), dict(cache=0), dict(masks=0), dict(workspace=0),
                                  dict(workspace=ON + 8), dict(q=ON + 8), dict(stride_cb=4), dict(cache_dtype=3),
                                  dict(cache_dtype=3, scale_page=ON, stride_cs=584), dict(block_table=_native.itab(None))])
def test_arguments_that_latent_attention_refuses(over):
    assert _native.library().eagle4_latent_attention(latent(**over), None) == NOT_COVERED
