"""Attention over the paged E4M3 cache: score factors beyond float32."""
import numpy as np
import pytest
import torch

from paged_cases import DEV, Cache, close
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("form", ["decode", "prompt"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_queries_of_zeros_before_scales_whose_product_float32_does_not_hold(form, dtype):
    """scale and the pages' scales are in their ranges, their product is not: scores of zero stay zero, every key counts the same."""
    cache = Cache([70, 300], 2, 128, 32, seed=22, scale_exponents=(2, 5))
    q = torch.zeros(2, 4 * 128, dtype=dtype)
    if form == "decode":
        got = K.paged_attention_decode_forward(q.to(DEV), *cache.device(), scale=2.0 ** 126)
    else:
        got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.arange(3, dtype=torch.int32, device=DEV), scale=2.0 ** 126)
    close(got, *cache.attention(q.view(-1, 4, 128).double().numpy(), np.arange(3), scale=1.0), dtype)
