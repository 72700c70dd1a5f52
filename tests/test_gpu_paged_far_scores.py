"""Attention over the paged E4M3 cache in fp16 where scores are far apart or far out: a weight never passes fp16's largest value."""
import numpy as np
import pytest
import torch

from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
DEV, HF = "cuda:0", torch.float16
F8 = torch.float8_e4m3fn


def _paged(keys, values, page, value_scale=1.0):
    """keys, values [kv_heads, positions, dim] (E4M3 values) of one sequence as a cache, its pages in order."""
    kv_heads, positions, dim = keys.shape
    pages = -(-positions // page)
    blank = torch.zeros(kv_heads, pages * page - positions, dim, device=DEV)
    keys, values = (torch.cat([t, blank], 1).view(kv_heads, pages, page, dim).transpose(0, 1) for t in (keys, values))
    return (keys.contiguous().to(F8), values.transpose(2, 3).contiguous().to(F8), torch.ones(pages, kv_heads, device=DEV), torch.full((pages, kv_heads), value_scale, device=DEV),
            torch.arange(pages, dtype=torch.int32, device=DEV)[None].contiguous(), torch.tensor([positions], dtype=torch.int32, device=DEV))


# (tokens, heads): the decode form; prompts in blocks of 128 and of 256 rows, the latter's earlier tokens without a position
@pytest.mark.parametrize("tokens,heads", [(1, 2), (70, 2), (560, 128)])
def test_scores_that_float32_holds_in_steps_of_sixteen(tokens, heads):
    """Scores of 2^27 + 16 and 2^27 + 32 (to base 2): the larger key has all the weight but 2^-16; a weight of 2^16 would be fp16's infinity."""
    scale = np.float32(0.6931472)
    assert np.float32(scale * np.float32(1.4426950408889634)) == 1.0
    keys, values = torch.zeros(1, 200, 64, device=DEV), torch.ones(1, 200, 64, device=DEV)
    keys[:, :, 0], keys[:, 20, 1], keys[:, 100, 1] = 256.0, 1.0, 2.0
    values[:, 100] = 3.0
    kp, vp, ks, vs, table, lengths = _paged(keys, values, 16)
    ks.fill_(16.0)
    q = torch.zeros(tokens, heads, 64, device=DEV)
    q[:, :, 0], q[:, :, 1] = 32768.0, 1.0
    q = q.view(tokens, -1).to(HF)
    if tokens == 1:
        got = K.paged_attention_decode_forward(q, kp, vp, ks, vs, table, lengths, scale=float(scale))
    else:
        cu = torch.tensor([0, tokens], dtype=torch.int32, device=DEV)
        got = K.paged_attention_prompt_forward(q, kp, vp, ks, vs, table, lengths, cu, scale=float(scale))
    assert bool(((got[-60:] - 3.0).abs() <= 3 * 2.0 ** -10).all()), got[-1, :4]
