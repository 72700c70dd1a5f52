"""Tree attention in blocks whose waves work in two ways (192 rows): queries that one half of a workgroup alone has to scale before the product, and calls repeated bit for bit."""
import numpy as np
import pytest
import torch

from oracle import tree_oracle as T
from paged_cases import DEV, Cache, close, queries
from pocketllm_amd import hip_kernel as K
from test_gpu_tree_attention import random_tree

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("rows", ["first", "last", "all"])
@pytest.mark.parametrize("nodes,heads,kv_heads,dim", [(64, 24, 8, 128), (150, 1, 1, 64), (192, 4, 4, 128)])
def test_large_queries_in_one_half_of_a_block(nodes, heads, kv_heads, dim, rows):
    """Queries around 2^120, whose products with codes pass the largest float32 before the pages' scales bring them back, in the rows that waves 0 to 3 have, in those of waves 4 to 7,
    in both; the others are around one beside them, so that their scores are none."""
    rng = np.random.default_rng(nodes)
    cache = Cache([2800 + nodes, 40 + nodes], kv_heads, dim, 32, seed=nodes, scale_exponents=(-125, -121))
    cache.value_scales = np.where(np.isnan(cache.value_scales), cache.value_scales, np.float32(2.0 ** -5)).astype(np.float32)
    parents = np.array(random_tree(rng, nodes) + random_tree(rng, nodes), dtype=np.int32)
    group, tokens = heads // kv_heads, 2 * nodes
    q = queries(tokens, heads, dim, BF, seed=1).view(tokens, heads, dim)
    row = (torch.arange(tokens)[:, None] % nodes * group + torch.arange(heads)[None] % group) % 192
    large = {"first": row < 128, "last": row >= 128, "all": row >= 0}[rows]
    q = torch.where(large[..., None], q * 2.0 ** 120, q).reshape(tokens, heads * dim)
    out = K.paged_attention_tree_forward(q.to(DEV), *cache.device(), torch.from_numpy(parents).to(DEV))
    torch.cuda.synchronize()
    assert large.any() and torch.isfinite(q.float()).all()
    want = T.tree_attention(q.double().numpy().reshape(tokens, heads, dim), cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales, cache.table, cache.lengths,
                            parents, np.array([0, nodes, tokens]), dim ** -0.5)
    close(out, *want, BF)


@pytest.mark.parametrize("nodes,pasts,heads,kv_heads,dim,dtype", [
    ([26] * 32, 900, 12, 2, 128, BF), ([70, 200, 0, 100], 3000, 8, 4, 64, torch.float16), ([64, 64], 2500, 24, 8, 128, BF), ([8], 700, 4, 4, 64, torch.float16),
])
def test_a_call_repeated_is_the_same_to_the_bit(nodes, pasts, heads, kv_heads, dim, dtype):
    rng = np.random.default_rng(heads)
    cache = Cache([int(p) + n for p, n in zip(rng.integers(0, pasts, len(nodes)), nodes)], kv_heads, dim, 64, seed=heads)
    q, device = queries(sum(nodes), heads, dim, dtype).to(DEV), cache.device()
    parents = torch.tensor(sum((random_tree(rng, n) if n else [] for n in nodes), []), dtype=torch.int32, device=DEV)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(nodes)]), dtype=torch.int32, device=DEV) if len(set(nodes)) > 1 else None
    first = K.paged_attention_tree_forward(q, *device, parents, cu_steps=cu)
    for _ in range(20):
        assert torch.equal(K.paged_attention_tree_forward(q, *device, parents, cu_steps=cu), first)
