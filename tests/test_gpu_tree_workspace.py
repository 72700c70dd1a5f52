"""The C entry of tree attention with exactly the workspace that it asks for, rows behind the last sequence among its rows: nothing outside of the output and the workspace is written."""
import numpy as np
import pytest
import torch

from oracle import tree_oracle as T
from paged_cases import DEV, Cache, close, queries
from pocketllm_amd import _ffi
from test_gpu_tree_attention import random_tree

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("seqs,nodes,past,heads,kv_heads,dim,tail", [
    (32, 26, 300, 3, 1, 64, 1), (32, 26, 300, 6, 1, 128, 70), (32, 70, 40, 4, 4, 64, 5), (31, 26, 300, 3, 1, 64, 3), (33, 20, 100, 4, 2, 64, 2), (63, 9, 200, 2, 1, 128, 4),
    (1, 90, 1000, 2, 1, 64, 9), (2, 200, 700, 1, 1, 128, 1), (64, 26, 100, 3, 1, 64, 3),
])
def test_rows_behind_the_last_sequence(seqs, nodes, past, heads, kv_heads, dim, tail):
    rng = np.random.default_rng(seqs + tail)
    sizes = [int(n) for n in rng.integers(1, nodes + 1, seqs)]
    cache = Cache([int(p) + n for p, n in zip(rng.integers(0, past + 1, seqs), sizes)], kv_heads, dim, 16, seed=seqs)
    cu = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    tokens = int(cu[-1]) + tail
    parents = np.array(sum((random_tree(rng, n) for n in sizes), []) + [0] * tail, dtype=np.int32)
    q = queries(tokens, heads, dim, BF, seed=2)
    lib, guard = _ffi.load_library(), 4096
    need = lib.pllm_paged_attention_tree_workspace_bytes(tokens, seqs, 0, heads, kv_heads, dim, cache.width * 16)
    assert need % 256 == 0 and (need > 0 or seqs >= 64)
    ws = torch.full((need + 2 * guard,), 0x55, dtype=torch.uint8, device=DEV)
    out = torch.full((guard + tokens * heads * dim + guard,), 7.0, dtype=BF, device=DEV)
    dev = [t.to(DEV) for t in (q, torch.from_numpy(parents), torch.from_numpy(cu))]
    kp, vp, ks, vs, table, lengths = cache.device()
    for _ in range(2):                                                        # (the second time beside what the first left)
        status = lib.pllm_paged_attention_tree(dev[0].data_ptr(), heads * dim, 2, kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), cache.pool, 16, table.data_ptr(),
                                               cache.width, cache.width, lengths.data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), tokens, seqs, heads, kv_heads, dim, dim ** -0.5,
                                               out[guard:].data_ptr(), ws[guard:].data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert status == 0
        torch.cuda.synchronize()
        assert bool((out[:guard] == 7).all()) and bool((out[-guard:] == 7).all()) and bool((ws[:guard] == 0x55).all()) and bool((ws[need + guard:] == 0x55).all())
        got = out[guard:-guard].view(tokens, heads * dim)
        assert not got[int(cu[-1]):].any()
    close(got, *T.tree_attention(q.double().numpy().reshape(tokens, heads, dim), cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales, cache.table, cache.lengths,
                                 parents, cu, dim ** -0.5), BF)
