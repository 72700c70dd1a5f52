"""Decode attention over the paged E4M3 cache: outputs that a wider table does not change."""
import numpy as np
import pytest
import torch

from paged_cases import DEV, Cache, close, queries
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dim,kv_heads,group,steps,dtype", [(128, 2, 6, 1, BF), (64, 4, 3, 2, HF), (128, 1, 8, 5, HF)])
def test_the_width_of_the_table_changes_no_bit(dim, kv_heads, group, steps, dtype):
    """Sequences of one to sixteen runs, and of more, before tables that have room for them and for many times as many."""
    lengths = [1, 900, 1030, 2049, 5000, 7900, 20, 9001]
    cache = Cache(lengths, kv_heads, dim, 64, seed=21, width=1100)
    kp, vp, ks, vs, table, held = cache.device()
    q = queries(len(lengths) * steps, kv_heads * group, dim, dtype, seed=4).view(len(lengths), steps, -1).to(DEV)
    together = K.paged_attention_decode_forward(q, kp, vp, ks, vs, table, held)
    for s, length in enumerate(lengths):
        for width in (-(-length // 64), 128, 150, 400):
            if 64 * width >= length:
                alone = K.paged_attention_decode_forward(q[s:s + 1], kp, vp, ks, vs, table[s:s + 1, :width], held[s:s + 1])
                assert torch.equal(alone[0], together[s]), (length, width)
    want, note = cache.attention(q.view(-1, kv_heads * group, dim).cpu().double().numpy(), np.arange(len(lengths) + 1) * steps)
    close(together, want, note, dtype)
