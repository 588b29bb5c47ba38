"""What latent verify attention refuses before any launch, beside the refusals of the sampled round's operators."""

import pytest
import torch

I32, BF16, FP8 = torch.int32, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("shape,error", [((3,), RuntimeError), ((3, 1), RuntimeError), ((5, 1), RuntimeError),  # a host tensor
                                         ((3, 2), ValueError), ((3, 0), ValueError), ((2, 1), ValueError), ((3, 1, 1), ValueError)])
def test_scales_are_one_a_page(shape, error):
    """Scales of several heads are not a latent cache's: the first head's would have been taken for all."""
    from eagle_harness.vllm.latent_attention import latent_verify_attention

    with pytest.raises(error):
        latent_verify_attention(
            torch.zeros(3, 4, 576, dtype=BF16), torch.zeros(3, 576, dtype=BF16), torch.zeros(3, 16, 576, dtype=FP8),
            torch.zeros(1, 2, dtype=I32), torch.zeros(1, dtype=I32), torch.tensor([0, 3], dtype=I32),
            torch.ones(1, 3, dtype=torch.int64), 0.1, torch.zeros(3, 4, 512, dtype=BF16), max_query_len=3,
            latent_scale=torch.ones(shape))
