"""paged_attention_tree_forward and the append of a tree's nodes against their float64 forms: shapes of trees, lengths, sizes of pages and groups, both kernels, masked
places that hold anything, offsets and tables that hold anything, other strides, streams and captured calls."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P, tree_oracle as T
from paged_cases import DEV, Cache, close, queries
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu


def random_tree(rng, n):
    return [-1] + [int(rng.integers(max(-1, i - 9), i)) for i in range(1, n)]


def check(cache, nodes, heads, dtype, parents, size=1.0, ragged=True, tail=0, seed=0, scale=None, device=None):
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    tokens = int(cu[-1]) + tail
    q = queries(tokens, heads, cache.dim, dtype, seed, size)
    parents = np.array(sum(parents, []) + [0] * tail, dtype=np.int32)
    out = K.paged_attention_tree_forward(q.to(DEV), *(device or cache.device()), torch.from_numpy(parents).to(DEV), cu_steps=torch.from_numpy(cu).to(DEV) if ragged else None, scale=scale)
    torch.cuda.synchronize()
    want = T.tree_attention(q.double().numpy().reshape(tokens, heads, cache.dim), cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales, cache.table, cache.lengths,
                            parents, cu, cache.dim ** -0.5 if scale is None else scale)
    assert not out[int(cu[-1]):].any()
    close(out, *want, dtype)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nodes,past,heads,kv_heads,dim,page", [
    (1, 0, 1, 1, 64, 16), (1, 63, 8, 2, 128, 64), (2, 1100, 6, 1, 128, 16), (8, 700, 4, 4, 64, 16), (13, 51, 12, 2, 64, 32), (26, 200, 6, 1, 128, 64), (26, 1500, 12, 2, 128, 128),
    (63, 1, 2, 2, 64, 16), (64, 64, 2, 1, 128, 32), (64, 1030, 8, 1, 64, 64), (65, 130, 1, 1, 64, 128), (100, 3, 16, 1, 64, 16), (200, 0, 3, 1, 128, 64), (256, 77, 2, 1, 64, 32),
])
def test_trees_of_all_sizes(nodes, past, heads, kv_heads, dim, page, dtype):
    rng = np.random.default_rng(nodes + past)
    cache = Cache([past + nodes] * 2, kv_heads, dim, page, seed=nodes)
    trees = [random_tree(rng, nodes) for _ in range(2)]
    a = check(cache, [nodes] * 2, heads, dtype, trees, ragged=False)
    b = check(cache, [nodes] * 2, heads, dtype, trees, ragged=True)
    assert a.shape == b.shape


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(6, 1, 128, 64), (4, 2, 64, 16), (16, 1, 64, 32)])
def test_ragged_trees(heads, kv_heads, dim, page):
    nodes = [1, 0, 40, 7, 64, 130, 2, 0]
    pasts = [0, 5, 1300, 15, 64, 700, 1025, 0]
    rng = np.random.default_rng(heads)
    cache = Cache([p + n for p, n in zip(pasts, nodes)], kv_heads, dim, page, seed=3)
    check(cache, nodes, heads, torch.bfloat16, [random_tree(rng, n) if n else [] for n in nodes], tail=3)


def test_many_sequences_of_few_nodes():
    rng = np.random.default_rng(5)
    nodes = [int(n) for n in rng.integers(0, 9, 70)]
    cache = Cache([int(p) + n for p, n in zip(rng.integers(0, 90, 70), nodes)], 1, 64, 16, seed=6, width=70)
    check(cache, nodes, 2, torch.float16, [random_tree(rng, n) if n else [] for n in nodes], tail=1)


@pytest.mark.parametrize("seqs,nodes,heads,dim,past,dtype", [
    (66, 26, 6, 128, 900, torch.bfloat16), (64, 12, 16, 64, 1000, torch.float16), (70, 80, 1, 64, 2000, torch.bfloat16), (65, 100, 3, 128, 64, torch.float16),
])
def test_many_sequences_of_many_rows(seqs, nodes, heads, dim, past, dtype):
    """64 sequences and more: blocks and halves of blocks in the order of the sequences, of the same number of nodes and of any."""
    rng = np.random.default_rng(seqs)
    cache = Cache([int(p) + nodes for p in rng.integers(0, past, seqs)], 1, dim, 64, seed=seqs)
    check(cache, [nodes] * seqs, heads, dtype, [random_tree(rng, nodes) for _ in range(seqs)], ragged=False)
    some = [int(n) for n in rng.integers(0, nodes + 1, seqs)]
    check(cache, some, heads, dtype, [random_tree(rng, n) if n else [] for n in some], tail=5)


@pytest.mark.parametrize("nodes,pasts,heads,kv_heads,dim,dtype", [
    ([70, 200, 0, 100, 5, 256], [3000, 700, 10, 0, 1900, 64], 32, 32, 64, torch.bfloat16),       # more units than run at once, some sequences in runs
    ([100, 30, 90], [900, 2500, 64], 48, 16, 128, torch.float16),
    ([70, 5], [300, 130], 260, 260, 64, torch.bfloat16),                      # more heads than compute units
    ([66], [100000], 1, 1, 64, torch.float16),                                # as many runs as a block has
    ([70, 66], [20000, 9], 2, 1, 128, torch.bfloat16),
])
def test_keys_cut_in_runs(nodes, pasts, heads, kv_heads, dim, dtype):
    rng = np.random.default_rng(heads)
    cache = Cache([p + n for p, n in zip(pasts, nodes)], kv_heads, dim, 64, seed=heads)
    check(cache, nodes, heads, dtype, [random_tree(rng, n) if n else [] for n in nodes], tail=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nodes,pasts,heads,kv_heads,dim", [
    (150, [0, 700, 63], 1, 1, 64), (129, [1000], 2, 2, 128), (100, [3000, 5, 130], 3, 1, 128), (192, [64, 64], 4, 4, 64), (64, [2500, 1], 24, 8, 128), (65, [40, 1500], 16, 2, 64),
])
def test_rows_that_fill_three_quarters_of_a_block(nodes, pasts, heads, kv_heads, dim, dtype):
    """129 to 192 rows, 257 to 384, 513 to 576: some waves have rows of their own, some share them."""
    rng = np.random.default_rng(nodes)
    cache = Cache([p + nodes for p in pasts], kv_heads, dim, 32, seed=nodes)
    trees = [random_tree(rng, nodes) for _ in pasts]
    check(cache, [nodes] * len(pasts), heads, dtype, trees, ragged=False)
    which = cache.table[0, 0]                                                 # a NaN among the keys of the past, one among the last node's values
    cache.key_codes[which, 0, 0, 1] = 0x7f
    last = pasts[-1] + nodes - 1
    cache.value_codes[cache.table[len(pasts) - 1, last // 32], kv_heads - 1, 9, last % 32] = 0xff
    check(cache, [nodes] * len(pasts), heads, dtype, trees, ragged=False, size=3.0)


@pytest.mark.parametrize("n", [10, 70])
def test_a_chain_is_the_causal_form(n):
    """The nodes one after the other: what the prompt and the decode form give, within both kernels' roundings against the float64 form."""
    cache = Cache([900 + n], 1, 128, 64, seed=1)
    check(cache, [n], 4, torch.bfloat16, [list(range(-1, n - 1))])
    cu = np.array([0, n])
    q = queries(n, 4, 128, torch.bfloat16)
    want = cache.attention(q.double().numpy().reshape(n, 4, 128), cu)
    out = K.paged_attention_tree_forward(q.to(DEV), *cache.device(), torch.arange(-1, n - 1, dtype=torch.int32, device=DEV))
    close(out, *want, torch.bfloat16)


@pytest.mark.parametrize("n,heads", [(20, 2), (90, 3)])
@pytest.mark.parametrize("parents", ["own", "behind", "far", "roots"])
def test_parents_that_are_no_earlier_node_are_none(n, heads, parents):
    tree = {"own": list(range(n)), "behind": [(i + 3) % (n + 7) if i % 2 else -1 for i in range(n)], "far": [-2**31, 2**31 - 1] * (n // 2), "roots": [-1] * n}[parents]
    check(Cache([130 + n], 1, 64, 32, seed=2), [n], heads, torch.float16, [tree])


@pytest.mark.parametrize("n,heads", [(24, 2), (90, 3)])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_nan_of_nodes_that_are_not_ancestors_stays_away(n, heads, where):
    """Codes of NaN in one node: the rows that descend from it are NaN (in its dimension, for a value), no other."""
    rng = np.random.default_rng(n)
    past, tree = 61, random_tree(rng, n)
    cache = Cache([past + n], 1, 64, 16, seed=4)
    for node in (1, n // 2, n - 1):
        at = past + node
        if where == "keys":
            cache.key_codes[cache.table[0, at // 16], 0, at % 16, 5] = 0x7f
        else:
            cache.value_codes[cache.table[0, at // 16], 0, 7, at % 16] = 0xff
    check(cache, [n], heads, torch.bfloat16, [tree])


@pytest.mark.parametrize("length", [-5, 0, 7, 30, 2**31 - 1])
@pytest.mark.parametrize("n", [12, 80])
def test_lengths_that_do_not_hold_the_tree(length, n):
    """Nodes without a place in the cache, or behind the table's end: what has none is seen by nobody."""
    cache = Cache([96], 1, 64, 16, seed=5)
    cache.lengths = np.array([length], dtype=np.int32)
    check(cache, [n], 2, torch.float16, [random_tree(np.random.default_rng(n), n)])


def test_table_entries_without_a_page_and_unordered_offsets():
    cache = Cache([200, 150], 1, 64, 16, seed=7)
    cache.table[0, 3], cache.table[0, 11], cache.table[1, 0] = -7, 2**30, cache.pool
    rng = np.random.default_rng(1)
    check(cache, [30, 9], 4, torch.bfloat16, [random_tree(rng, 30), random_tree(rng, 9)])
    # offsets that fall or pass the rows: no fault, and rows of no sequence are zeros
    q, parents = queries(39, 4, 64, torch.bfloat16).to(DEV), torch.zeros(39, dtype=torch.int32, device=DEV)
    for cu in ([0, 50, 20], [0, -3, 39], [0, 2**31 - 1, -2**31], [7, 7, 7]):
        out = K.paged_attention_tree_forward(q, *cache.device(), parents, cu_steps=torch.tensor(cu, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        assert out.shape == q.shape


def test_more_nodes_than_a_tree_can_have_are_zeros():
    cache = Cache([300, 90], 1, 64, 64, seed=8)
    rng = np.random.default_rng(2)
    out = check(cache, [257, 40], 1, torch.float16, [random_tree(rng, 257), random_tree(rng, 40)])
    assert not out[:257].any() and out[257:].any()


def test_slices_of_a_wider_projection_and_tables():
    cache, n = Cache([300, 280], 2, 64, 32, seed=9), 18
    rng = np.random.default_rng(3)
    trees = [random_tree(rng, n) for _ in range(2)]
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device=DEV)
    q = queries(2 * n, 4, 64, torch.bfloat16).to(DEV)
    device = list(cache.device())
    want = K.paged_attention_tree_forward(q, *device, parents)
    wide = torch.full((2 * n, 700), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 64:320] = q
    device[4] = torch.cat([device[4], torch.full((2, 3), 2**30, dtype=torch.int32, device=DEV)], 1)[:, :device[4].size(1)]
    assert torch.equal(K.paged_attention_tree_forward(wide[:, 64:320], *device, parents), want)
    odd = torch.empty(2 * n * 256 + 3, dtype=torch.bfloat16, device=DEV)[3:].view(2 * n, 256).copy_(q)   # (not on 16 bytes: copied)
    assert torch.equal(K.paged_attention_tree_forward(odd, *device, parents), want)


def test_a_sequence_does_not_depend_on_its_batch():
    n, rng = 12, np.random.default_rng(4)
    trees = [random_tree(rng, n) for _ in range(5)]
    cache = Cache([1500, 40, 3000, 700, 2100], 1, 128, 64, seed=10)
    q = queries(5 * n, 4, 128, torch.bfloat16).to(DEV)
    device = cache.device()
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device=DEV)
    every = K.paged_attention_tree_forward(q, *device, parents).view(5, n, -1)
    for s in (0, 2, 4):
        alone = K.paged_attention_tree_forward(q[s * n:(s + 1) * n], *device[:4], device[4][s:s + 1], device[5][s:s + 1], parents[s * n:(s + 1) * n])
        assert torch.equal(alone, every[s])


@pytest.mark.parametrize("n", [10, 90])
def test_captured_and_replayed_on_two_streams(n):
    """One graph per shape, replayed on other queries, trees and lengths, beside eager calls on another stream; every replay against the eager call."""
    cache = Cache([1200] * 2, 1, 128, 64, seed=11)
    device = list(cache.device())
    rng = np.random.default_rng(5)
    q = queries(2 * n, 6, 128, torch.bfloat16).to(DEV)
    parents = torch.tensor(random_tree(rng, n) + random_tree(rng, n), dtype=torch.int32, device=DEV)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.paged_attention_tree_forward(q, *device, parents)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = K.paged_attention_tree_forward(q, *device, parents)
    for i in range(4):
        q.copy_(queries(2 * n, 6, 128, torch.bfloat16, seed=i))
        parents.copy_(torch.tensor(random_tree(rng, n) + random_tree(rng, n), dtype=torch.int32))
        device[5].copy_(torch.tensor([1200 - 40 * i, 100 + n + 300 * i], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            want = K.paged_attention_tree_forward(q, *device, parents)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("heads,tokens", [(8, 2), (2, 60), (16, 40)])
def test_appended_nodes_are_turned_by_their_depth(heads, tokens):
    """The append with positions against the same call at those places of a cache of its own: the same codes, scales and queries."""
    dim, kv_heads, page, past = 64, 2, 16, 21
    depths = np.array([0] + list(np.random.default_rng(6).integers(1, 6, tokens - 1)), dtype=np.int32)
    cache = Cache([past + tokens], kv_heads, dim, page, seed=12)
    cos, sin = P.rotary_rows(past + 8, dim, 32)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(tokens, n * dim, generator=g).to(torch.bfloat16) for n in (heads, kv_heads, kv_heads))
    positions = np.concatenate([past + depths])
    device = cache.device()
    turned = K.paged_kv_append_forward(q.to(DEV), k.to(DEV), v.to(DEV), *device, cos_table=torch.from_numpy(cos).to(DEV), sin_table=torch.from_numpy(sin).to(DEV), rope_dim=32,
                                       positions=torch.from_numpy(positions).to(DEV))
    torch.cuda.synchronize()
    keys = P.turn(k.double().numpy().reshape(tokens, kv_heads, dim), cos[positions], sin[positions], 32)
    want = P.append(keys, v.double().numpy().reshape(tokens, kv_heads, dim), cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales, cache.table, cache.lengths,
                    np.array([0, tokens]))
    for s in range(past + tokens):
        which, slot = cache.table[0, s // page], s % page
        assert np.array_equal(P.e4m3_decode(device[0].view(torch.uint8)[which, :, slot].cpu().numpy()), want[0][which, :, slot], equal_nan=True)
        assert np.array_equal(P.e4m3_decode(device[1].view(torch.uint8)[which, :, :, slot].cpu().numpy()), want[1][which, :, :, slot], equal_nan=True)
    rows = P.turn(q.double().numpy().reshape(tokens, heads, dim), cos[positions], sin[positions], 32)
    got = turned.cpu().double().numpy().reshape(tokens, heads, dim)
    # a product, a fused product and sum in float32 (half a step of 2^-23 each of the magnitudes), one rounding to bf16
    size = np.abs(q.double().numpy().reshape(tokens, heads, dim)).max() * 2
    assert (np.abs(got - rows) <= 2.0 ** -8 * np.abs(rows) + 2 * 2.0 ** -24 * size * (1 + 2.0 ** -8)).all()
    # positions outside the tables are the nearest row, not a fault
    far = torch.full((tokens,), 2**31 - 1, dtype=torch.int32, device=DEV)
    near = torch.full((tokens,), past + 7, dtype=torch.int32, device=DEV)
    a, b = (K.paged_kv_append_forward(q.to(DEV), k.to(DEV), v.to(DEV), *cache.device(), cos_table=torch.from_numpy(cos).to(DEV), sin_table=torch.from_numpy(sin).to(DEV), rope_dim=32,
                                      positions=p) for p in (far, near))
    assert torch.equal(a, b)


def test_positions_are_refused():
    cache = Cache([20], 1, 64, 16)
    k = torch.zeros(2, 64, dtype=torch.float16, device=DEV)
    for positions in (torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="positions must be"):
            K.paged_kv_append_forward(None, k, k, *cache.device(), positions=positions)
