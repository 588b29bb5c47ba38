"""What the sampled round's operators refuse, before any launch and on the CPU: arguments that do not fit raise ValueError,
layouts and types that the kernels do not address raise NotCovered, host tensors that pass are refused by the launch."""

import pytest
import torch

from eagle_harness.kernels._native import NotCovered

I32 = torch.int32


class Store:
    def __init__(self, slots=2, width=4):
        self.width = width
        self.path = torch.zeros(slots, width, dtype=I32)
        self.path_len = torch.ones(slots, dtype=I32)


def sample(**over):
    from eagle_harness.vllm.tree_accept import sample_tree

    x = dict(logits=torch.zeros(4, 10), drafted=torch.zeros(4, dtype=torch.int64), cu=torch.tensor([0, 4], dtype=I32),
             slots=torch.zeros(1, dtype=I32), parents=torch.zeros(2, 4, dtype=I32), store=Store(), coins=torch.zeros(4),
             final=torch.zeros(1), temperature=torch.ones(1), probs=None)
    x.update(over)
    return sample_tree(x["logits"], x["drafted"], x["cu"], x["slots"], x["parents"], x["store"], x["coins"], x["final"],
                       x["temperature"], draft_probs=x["probs"])


@pytest.mark.parametrize("over,error", [
    (dict(logits=torch.zeros(40)), ValueError),
    (dict(probs=torch.zeros(4, 9)), ValueError),
    (dict(probs=torch.zeros(3, 10)), ValueError),
    (dict(logits=torch.zeros(10, 4).t()), NotCovered),
    (dict(logits=torch.zeros(4, 10, dtype=torch.float64)), NotCovered),
    (dict(logits=torch.zeros(4, 10, dtype=torch.int64)), NotCovered),
    (dict(store=Store(width=65), parents=torch.zeros(2, 65, dtype=I32)), NotCovered),
    (dict(drafted=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(drafted=torch.zeros(4)), NotCovered),
    (dict(parents=torch.zeros(2, 3, dtype=I32)), ValueError),
    (dict(coins=torch.zeros(3)), ValueError),
    (dict(coins=torch.zeros(4, dtype=torch.float64)), ValueError),
    (dict(coins=torch.zeros(8)[::2]), ValueError),
    (dict(final=torch.zeros(0)), ValueError),
    (dict(temperature=torch.ones(1, dtype=torch.int64)), ValueError),
    (dict(), RuntimeError),  # a host tensor
])
def test_sample_tree(over, error):
    with pytest.raises(error):
        sample(**over)


def pages(heads=2, dim=8, blocks=3, page=4):
    return torch.zeros(blocks, page, heads, dim, dtype=torch.float8_e4m3fn), torch.ones(blocks, heads)


def write(**over):
    from eagle_harness.vllm.kv_pages import write_kv_pages

    cache, scale = pages()
    x = dict(key=torch.zeros(4, 2, 8), value=torch.zeros(4, 2, 8), key_cache=cache, value_cache=cache.clone(), k_scale=scale,
             v_scale=scale.clone(), table=torch.zeros(1, 2, dtype=I32), context=torch.zeros(1, dtype=I32),
             starts=torch.tensor([0, 4], dtype=I32), idx=None, path=None, path_len=None)
    x.update(over)
    return write_kv_pages(x["key"], x["value"], x["key_cache"], x["value_cache"], x["k_scale"], x["v_scale"], x["table"],
                          x["context"], x["starts"], max_query_len=4, idx_mapping=x["idx"], path=x["path"],
                          path_len=x["path_len"])


@pytest.mark.parametrize("over,error", [
    (dict(value=None), ValueError),
    (dict(v_scale=None), ValueError),
    (dict(key=torch.zeros(4, 16)), ValueError),
    (dict(value=torch.zeros(4, 2, 7)), ValueError),
    (dict(value=torch.zeros(4, 2, 8, dtype=torch.bfloat16)), NotCovered),
    (dict(key=torch.zeros(4, 3, 8), value=torch.zeros(4, 3, 8)), ValueError),
    (dict(key=torch.zeros(4, 8, 2).transpose(1, 2)), NotCovered),
    (dict(key_cache=torch.zeros(3, 4, 2, 8, dtype=torch.uint8)), NotCovered),
    (dict(k_scale=torch.ones(2, 2)), ValueError),
    (dict(k_scale=torch.ones(3, 2, dtype=torch.float64)), ValueError),
    (dict(k_scale=torch.ones(1, 1).expand(3, 2)), ValueError),
    (dict(v_scale=torch.ones(3, 1).expand(3, 2)), ValueError),
    (dict(table=torch.zeros(2, dtype=I32)), ValueError),
    (dict(table=torch.zeros(0, 2, dtype=I32)), ValueError),
    (dict(context=torch.zeros(0, dtype=I32)), ValueError),
    (dict(context=torch.zeros(1)), NotCovered),
    (dict(path=torch.zeros(1, 4, dtype=I32)), ValueError),
    (dict(path=torch.zeros(1, 4, dtype=I32), path_len=torch.ones(1, dtype=I32)), ValueError),
    (dict(path=torch.zeros(1, 4, dtype=I32), path_len=torch.ones(1, dtype=I32), idx=torch.zeros(0, dtype=I32)), ValueError),
    (dict(), RuntimeError),
])
def test_write_kv_pages(over, error):
    with pytest.raises(error):
        write(**over)


@pytest.mark.parametrize("over,error", [
    (dict(out=torch.zeros(4, 2, 8, dtype=torch.float64)), NotCovered),
    (dict(out=torch.zeros(4, 2, 9)), ValueError),
    (dict(table=torch.zeros(0, 2, dtype=I32)), ValueError),
    (dict(), RuntimeError),
])
def test_read_kv_pages(over, error):
    from eagle_harness.vllm.kv_pages import read_kv_pages

    cache, scale = pages()
    x = dict(out=torch.zeros(4, 2, 8), table=torch.zeros(1, 2, dtype=I32))
    x.update(over)
    with pytest.raises(error):
        read_kv_pages(cache, None, scale, None, x["table"], torch.tensor([0, 4], dtype=I32), x["out"], None, max_len=4)


BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("over,error", [
    (dict(q=torch.zeros(3, 576, dtype=BF16)), ValueError),
    (dict(new=torch.zeros(2, 576, dtype=BF16)), ValueError),
    (dict(cache=torch.zeros(3, 16, 512, dtype=BF16)), ValueError),
    (dict(out=torch.zeros(3, 4, 576, dtype=BF16)), ValueError),
    (dict(out=torch.zeros(3, 4, 512)), NotCovered),
    (dict(q=torch.zeros(3, 4, 576), new=torch.zeros(3, 576), out=torch.zeros(3, 4, 512),
          cache=torch.zeros(3, 16, 576)), NotCovered),
    (dict(cache=torch.zeros(3, 16, 576, dtype=torch.float16)), NotCovered),
    (dict(cache=torch.zeros(3, 16, 576, dtype=FP8)), ValueError),
    (dict(cache=torch.zeros(3, 16, 576, dtype=FP8), page_scale=torch.ones(2)), ValueError),
    (dict(cache=torch.zeros(3, 16, 576, dtype=FP8), page_scale=torch.ones(3, dtype=BF16)), ValueError),
    (dict(table=torch.zeros(1, 2, dtype=torch.int64)), NotCovered),
    (dict(masks=torch.zeros(1, 3, dtype=I32)), NotCovered),
    (dict(masks=torch.zeros(1, 2, dtype=torch.int64)), ValueError),
    (dict(masks=torch.zeros(0, 3, dtype=torch.int64)), ValueError),
    (dict(context=torch.zeros(0, dtype=I32)), ValueError),
    (dict(new=torch.zeros(576, 3, dtype=BF16).t()), NotCovered),
    (dict(width=65, masks=torch.zeros(1, 65, dtype=torch.int64)), NotCovered),
    (dict(q=torch.zeros(3, 4, 580, dtype=BF16)[..., :576]), NotCovered),  # rows not on 16 bytes
    (dict(q=torch.zeros(3, 4, 448, dtype=BF16), new=torch.zeros(3, 448, dtype=BF16), cache=torch.zeros(3, 16, 448, dtype=BF16),
          out=torch.zeros(3, 4, 384, dtype=BF16)), NotCovered),
    (dict(), RuntimeError),
])
def test_latent_verify_attention(over, error):
    from eagle_harness.vllm.latent_attention import latent_verify_attention

    x = dict(q=torch.zeros(3, 4, 576, dtype=BF16), new=torch.zeros(3, 576, dtype=BF16), cache=torch.zeros(3, 16, 576, dtype=BF16),
             table=torch.zeros(1, 2, dtype=I32), context=torch.zeros(1, dtype=I32), starts=torch.tensor([0, 3], dtype=I32),
             masks=torch.ones(1, 3, dtype=torch.int64), out=torch.zeros(3, 4, 512, dtype=BF16), width=3, page_scale=None)
    x.update(over)
    with pytest.raises(error):
        latent_verify_attention(x["q"], x["new"], x["cache"], x["table"], x["context"], x["starts"], x["masks"], 0.1, x["out"],
                                max_query_len=x["width"], latent_scale=x["page_scale"])


def test_the_library_refuses_what_reaches_it():
    """The C entries' own checks (status -1), for callers that bind them directly."""
    from eagle_harness.kernels import _native

    lib = _native.library()
    table = torch.zeros(4, 4, dtype=I32)
    tab = _native.itab(table)
    common = dict(q=16, latent_new=16, cache=16, out=16, workspace=16, workspace_bytes=1 << 40, block_table=tab,
                  context_lens=tab, query_start_loc=tab, masks=16, num_reqs=1, heads=16, rank=512, rope=64, page=16,
                  max_query_len=1, max_blocks=4, num_blocks=4)
    assert lib.eagle4_latent_attention_workspace(_native.LatentAttnArgs(**common)) > 0
    for over in (dict(rank=384), dict(rope=32), dict(max_query_len=0), dict(max_query_len=65), dict(heads=0), dict(page=0),
                 dict(dtype=2), dict(cache_dtype=1), dict(cache_dtype=3), dict(stride_qt=4), dict(q=8), dict(masks=0),
                 dict(page=1 << 30)):
        args = _native.LatentAttnArgs(**{**common, **over})
        assert lib.eagle4_latent_attention_workspace(args) == -1, over
        assert lib.eagle4_latent_attention(args, None) == -1, over
    assert lib.eagle4_latent_attention(_native.LatentAttnArgs(**{**common, "workspace_bytes": 16}), None) == -1
    assert lib.eagle4_latent_attention(_native.LatentAttnArgs(**{**common, "num_reqs": 0}), None) == 0
    sampled = dict(logits=16, drafted=tab, cu_num_logits=tab, idx_mapping=tab, parents=tab, coins=16, final_coins=16,
                   temperature=16, sampled=16, num_sampled=16, path=16, path_len=16, rows=4, num_reqs=1, width=4, vocab=9, slots=4)
    for over in (dict(width=0), dict(width=65), dict(vocab=0), dict(logits=0), dict(coins=0), dict(dtype=3), dict(slots=0),
                 dict(probs=16, prob_dtype=4)):
        assert lib.eagle4_sample_tree(_native.SampleTreeArgs(**{**sampled, **over}), None) == -1, over
    assert lib.eagle4_sample_tree(_native.SampleTreeArgs(**{**sampled, "num_reqs": 0}), None) == 0
    kv = dict(key=16, key_cache=16, k_scale=16, block_table=tab, context_lens=tab, query_start_loc=tab, tokens=4, num_reqs=1,
              heads=1, dim=8, page=4, max_blocks=2, num_blocks=2, max_rows=4)
    for over in (dict(key=0), dict(k_scale=0), dict(heads=0), dict(dim=0), dict(page=0), dict(dtype=3), dict(value=16),
                 dict(path=tab), dict(num_reqs=70000)):
        assert lib.eagle4_write_kv_pages(_native.WriteKvArgs(**{**kv, **over}), None) == -1, over
    assert lib.eagle4_write_kv_pages(_native.WriteKvArgs(**{**kv, "max_rows": 0}), None) == 0
    kv = {k: v for k, v in kv.items() if k not in ("context_lens", "query_start_loc", "max_rows")} | dict(start_loc=tab, max_len=4)
    for over in (dict(key=0), dict(num_blocks=-1), dict(dtype=5), dict(value=16), dict(num_reqs=70000)):
        assert lib.eagle4_read_kv_pages(_native.ReadKvArgs(**{**kv, **over}), None) == -1, over
    assert lib.eagle4_read_kv_pages(_native.ReadKvArgs(**{**kv, "max_len": 0}), None) == 0


def test_capacities_near_the_positions_limit():
    """Tables whose pages reach up to 2^31 positions leave no room for the tiles that are looked up ahead."""
    from eagle_harness.kernels import _native

    lib, tab = _native.library(), _native.itab(torch.zeros(4, 4, dtype=I32))
    args = dict(q=16, latent_new=16, cache=16, out=16, workspace=16, workspace_bytes=1 << 40, block_table=tab, context_lens=tab,
                query_start_loc=tab, masks=16, num_reqs=1, heads=16, rank=512, rope=64, max_query_len=1, num_blocks=4)
    for page, blocks, ok in ((1 << 16, (1 << 15) - 1, True), (1, (1 << 31) - 2049, True), (1, (1 << 31) - 2048, False),
                             (1 << 16, 1 << 15, False)):
        need = lib.eagle4_latent_attention_workspace(_native.LatentAttnArgs(**args, page=page, max_blocks=blocks))
        assert (need > 0) == ok, (page, blocks)
