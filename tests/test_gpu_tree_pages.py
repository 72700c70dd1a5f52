"""draft_tree_accept_forward, paged_cache_compact_forward and paged_cache_fork_forward against their plain forms: whole numbers, codes and scales are equal."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P, tree_oracle as T
from paged_cases import DEV, Cache
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


# ---- the accepted path ------------------------------------------------------------------------------------------------

def random_drafts(rng, nodes, alphabet=4):
    """Trees whose sampled tokens often follow an edge; children of one node may have the same token."""
    parents, drafted, sampled = [], [], []
    for n in nodes:
        parents += [-1] + [int(rng.integers(0, i)) for i in range(1, n)] if n else []
        drafted += list(rng.integers(0, alphabet, n))
        sampled += list(rng.integers(0, alphabet, n))
    return np.array(parents, dtype=np.int32), np.array(drafted, dtype=np.int64), np.array(sampled, dtype=np.int64)


def check_accept(nodes, parents, drafted, sampled, lengths, most=None, even=False):
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    got = K.draft_tree_accept_forward(torch.from_numpy(parents).to(DEV), torch.from_numpy(drafted).to(DEV), torch.from_numpy(sampled).to(DEV), ints(lengths),
                                      cu_steps=None if even else ints(cu), most=most)
    torch.cuda.synchronize()
    want = T.accept(parents, drafted, sampled, lengths, cu, got[0].size(1))
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)
    return got


@pytest.mark.parametrize("nodes", [[1], [26], [5, 0, 64, 65, 1, 130], [256, 255, 3], [2] * 70])
@pytest.mark.parametrize("alphabet", [1, 2, 5])
def test_paths(nodes, alphabet):
    rng = np.random.default_rng(len(nodes) + alphabet)
    for most in (None, 1, 3, 64, 65):
        check_accept(nodes, *random_drafts(rng, nodes, alphabet), rng.integers(0, 1000, len(nodes)) + np.array(nodes), most)
    if len(set(nodes)) == 1:
        check_accept(nodes, *random_drafts(rng, nodes, alphabet), np.array(nodes) + 7, None, even=True)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 129, 256])
def test_chains_to_their_end(n):
    """The longest paths: every node follows."""
    chain = np.arange(-1, n - 1, dtype=np.int32)
    tokens = np.arange(n, dtype=np.int64) + (1 << 40)                         # (tokens need all 64 bits compared)
    got = check_accept([n], chain, tokens, tokens + 1, [n + 5])
    assert got[1].item() == n and got[3].item() == n + 5
    check_accept([n], chain, tokens, tokens + 1 + (1 << 32), [n + 5])


def test_parents_and_offsets_that_hold_anything():
    rng = np.random.default_rng(9)
    parents, drafted, sampled = random_drafts(rng, [40], 2)
    parents[[3, 7, 9, 20]] = [2**31 - 1, -2**31, 39, 20]
    check_accept([40], parents, drafted, sampled, [40])
    for cu in ([0, 90, 20], [0, -3, 40], [0, 2**31 - 1, -2**31]):
        kept, counts, _, _ = K.draft_tree_accept_forward(torch.from_numpy(parents).to(DEV), torch.from_numpy(drafted).to(DEV), torch.from_numpy(sampled).to(DEV), ints([5, 6]), cu_steps=ints(cu))
        torch.cuda.synchronize()
        assert bool((counts >= 0).all()) and bool((counts <= 40).all()) and bool((kept < 40).all())
    big = random_drafts(rng, [300], 1)                                        # nodes behind the 256th are not looked at
    check_accept([300], *big, [300])
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    kept, counts, token, news = K.draft_tree_accept_forward(empty, empty.long(), empty.long(), ints([4, 9]), cu_steps=ints([0, 0, 0]), most=3)
    assert kept.tolist() == [[-1] * 3] * 2 and counts.tolist() == [0, 0] and token.tolist() == [-1, -1] and news.tolist() == [4, 9]


# ---- the move in the cache --------------------------------------------------------------------------------------------

def check_compact(caches, kept, counts, steps, cu=None):
    """caches share table and lengths.  Codes and scales of everything afterwards are the plain form's."""
    device = [c.device() for c in caches]
    table, lengths = device[0][4], device[0][5]
    K.paged_cache_compact_forward([d[:4] for d in device], table, lengths, ints(kept), ints(counts), cu if cu is not None else int(steps[0]))
    torch.cuda.synchronize()
    for c, d in zip(caches, device):
        with np.errstate(invalid="ignore", divide="ignore"):
            want = T.compact(c.key_codes, c.value_codes, c.key_scales, c.value_scales, c.table, c.lengths, np.asarray(kept), np.asarray(counts), steps)
        assert np.array_equal(P.e4m3_decode(d[0].view(torch.uint8).cpu().numpy()), want[0], equal_nan=True)
        assert np.array_equal(P.e4m3_decode(d[1].view(torch.uint8).cpu().numpy()), want[1], equal_nan=True)
        assert np.array_equal(d[2].cpu().numpy().astype(np.float64), want[2], equal_nan=True) and np.array_equal(d[3].cpu().numpy().astype(np.float64), want[3], equal_nan=True)
    return device


def random_path(rng, n, most):
    if n == 0:
        return [-1] * most, 0
    count = int(rng.integers(0, min(n, most) + 1))
    return sorted(rng.permutation(n)[:count].tolist()) + [-1] * (most - count), count


@pytest.mark.parametrize("kv_heads,dim,page", [(1, 64, 16), (2, 128, 64), (3, 64, 32), (2, 128, 128), (2, 64, 16)])
def test_random_paths(kv_heads, dim, page):
    rng = np.random.default_rng(page + dim)
    nodes = [1, 26, 64, 0, 200, 13, 256, 40]
    pasts = [0, 15, 16, 30, 3, 127, 64, 500]
    lengths = [p + n for p, n in zip(pasts, nodes)]
    first = Cache(lengths, kv_heads, dim, page, seed=1, scale_exponents=(-9, -2))
    second = Cache(lengths, kv_heads, dim, page, seed=1, scale_exponents=(-9, -2))
    second.key_codes[:], second.value_codes[:] = first.key_codes[:, ::-1], first.value_codes[:, :, ::-1]
    second.key_scales[:] = first.value_scales
    paths = [random_path(rng, n, 256) for n in nodes]
    check_compact([first, second], [p for p, _ in paths], [c for _, c in paths], nodes, ints(np.concatenate([[0], np.cumsum(nodes)])))


@pytest.mark.parametrize("past", [0, 5, 15, 16])
def test_even_trees_and_paths_that_stay(past):
    """A path of the first nodes moves nothing, not a code nor a scale; one that skips a node does."""
    cache = Cache([past + 20] * 2, 2, 64, 16, seed=2)
    device = check_compact([cache], [list(range(6))] * 2, [6, 3], [20, 20])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(device[0][:2], cache.device()[:2]))
    check_compact([cache], [[0, 1, 3, 4, 18, 19], [1, 2, 5, 9, -1, -1]], [6, 4], [20, 20])


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 128)])
def test_paths_of_several_stretches(dim, page):
    """Long paths, whole or with one node or every few left out, at borders of 64 tokens, behind pasts that end anywhere in a page."""
    kept = [list(range(1, 65)), [0] + list(range(2, 66)), list(range(100, 228)), [*range(63), *range(64, 130)], list(range(1, 256)), list(range(256)), list(range(0, 256, 3)), list(range(191, 256))]
    pasts = [0, 7, 16, 61, 64, 100, 129, 15]
    cache = Cache([p + 256 for p in pasts], 2, dim, page, seed=page, scale_exponents=(-9, -2))
    check_compact([cache], [k + [-1] * (256 - len(k)) for k in kept], [len(k) for k in kept], [256] * 8)


def test_paths_that_are_none_and_places_without_a_page():
    cache = Cache([60, 60, 60, 60], 1, 64, 16, seed=3)
    cache.table[1, 2], cache.table[2, 1], cache.table[3, 3] = -1, 2**30, cache.pool
    kept = [[0, 3, 3, 9], [1, 30, 33, 39], [2, 17, 20, 35], [5, 9, 38, 40]]   # stops rising; sources and destinations without a page; leaves the tree
    check_compact([cache], kept, [4, 4, 4, 4], [40] * 4)
    check_compact([cache], kept, [2**31 - 1, -5, 0, 3], [40] * 4)
    check_compact([cache], [[-1, 2, 3, 4], [2**31 - 1, 3, 4, 5], [-2**31, 1, 2, 3], [3, 1, 2, 9]], [4] * 4, [40] * 4)
    for length in (-2**31, 0, 3, 39, 2**31 - 1):
        cache.lengths[:] = length
        check_compact([cache], kept, [4] * 4, [40] * 4)
    cache.lengths[:] = 60
    for cu in ([0, 40, 10, 2**31 - 1, -2**31], [-9, -3, 40, 300, 340], [0, 257, 257, 297, 297]):
        got = np.maximum(np.array(cu, dtype=np.int64), 0)
        got[0] = 0
        check_compact([cache], kept, [4] * 4, got[1:] - got[:-1], ints(cu))


def test_nan_codes_stay_nan_and_small_codes_round_to_even():
    cache = Cache([40], 1, 64, 16, seed=4)
    for p in range(3):
        cache.key_codes[cache.table[0, p], 0] = (np.arange(16 * 64) * 7 % 256).reshape(16, 64)
        cache.value_codes[cache.table[0, p], 0] = (np.arange(16 * 64) * 11 % 256).reshape(64, 16)
        cache.key_scales[cache.table[0, p]], cache.value_scales[cache.table[0, p]] = 2.0 ** (p * 2), 2.0 ** (3 - p * 3)
    check_compact([cache], [[0, 1, 9, 20, 21, 30]], [6], [32])


def test_more_layers_than_a_launch_holds():
    lengths, layers = [30, 21], []
    base = Cache(lengths, 1, 64, 16, seed=5)
    for i in range(67):
        c = Cache(lengths, 1, 64, 16, seed=5)
        c.key_codes, c.value_codes = np.roll(base.key_codes, i, axis=-1).copy(), np.roll(base.value_codes, i, axis=2).copy()
        layers.append(c)
    check_compact(layers, [[0, 2, 7, 11], [1, 3, 9, -1]], [4, 3], [12, 12])


# ---- the sequences of the next step -----------------------------------------------------------------------------------

def check_fork(cache, uses, sources, kept, reserve, layers=2):
    device = [cache.device() for _ in range(layers)]
    before = [[t.clone() for t in d[:4]] for d in device]
    got = K.paged_cache_fork_forward([d[:4] for d in device], device[0][4], ints(uses), ints(sources), ints(kept), ints(reserve))
    torch.cuda.synchronize()
    *want, copies = T.fork(cache.table, uses, sources, kept, reserve, cache.page)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)
    for d, b in zip(device, before):
        for t, old in zip(d[:4], b):
            for src, dst in copies:
                old[dst] = old[src]
            assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))
    return got, copies


def uses_of(cache, extra=()):
    uses = np.zeros(cache.pool, dtype=np.int64)
    for p in cache.table.reshape(-1):
        if 0 <= p < cache.pool:
            uses[p] += 1
    for p in extra:
        uses[p] += 1
    return uses


@pytest.mark.parametrize("kv_heads,dim,page", [(1, 64, 16), (2, 128, 64), (8, 128, 128), (3, 64, 32)])
def test_random_forks(kv_heads, dim, page):
    rng = np.random.default_rng(page)
    for trial in range(6):
        lengths = [int(n) for n in rng.integers(1, 400, 5)]
        cache = Cache(lengths, kv_heads, dim, page, seed=trial, spare=12, width=30)
        cache.table[cache.table >= cache.pool] = -1
        rows = int(rng.integers(1, 9))
        sources = rng.integers(-1, 5, rows)
        kept = [0 if s < 0 else int(rng.integers(0, lengths[s] + 1)) for s in sources]
        reserve = [k + int(rng.integers(0, 60)) for k in kept]
        uses = uses_of(cache, rng.integers(0, cache.pool, 2) if trial % 2 else ())
        check_fork(cache, uses, sources, kept, reserve, layers=1 + trial % 3)


def test_one_source_many_times():
    cache = Cache([40, 70], 2, 64, 16, seed=1, spare=20, width=8)
    cache.table[cache.table >= cache.pool] = -1
    got, copies = check_fork(cache, uses_of(cache), [0] * 6, [40] * 6, [41] * 6)
    assert len(copies) == 5 and got[1][int(cache.table[0, 0])].item() == 6    # five copies of the page in part, whole ones shared six times
    got, copies = check_fork(cache, uses_of(cache), [1, 1, 0, 0], [64, 64, 33, 30], [64, 80, 33, 46])
    assert len(copies) == 1                                                   # 64 tokens are whole pages; 30 end in the second page, which is whole for the row of 33
    _, copies = check_fork(cache, uses_of(cache), [0, 0], [40, 20], [40, 20])
    assert len(copies) == 1                                                   # the page that the second stops in is whole for the first
    _, copies = check_fork(cache, uses_of(cache, [cache.table[0, 2]]), [0, 1], [40, 70], [40, 70])
    assert len(copies) == 1                                                   # another holder has the page


def test_too_few_free_pages_and_everything_freed():
    cache = Cache([40, 70], 1, 64, 16, seed=2, spare=2, width=8)
    cache.table[cache.table >= cache.pool] = -1
    got, _ = check_fork(cache, uses_of(cache), [0, 0, 1], [40, 40, 70], [60, 60, 120])
    assert got[2].sum().item() > 0 and bool((got[0] >= -1).all())
    got, _ = check_fork(cache, uses_of(cache), [-1], [0], [0])
    assert not got[1].any() and bool((got[0] == -1).all())
    device = cache.device()
    table, uses, missing = K.paged_cache_fork_forward([device[:4]], device[4], ints(uses_of(cache)), ints([]), ints([]), ints([]))
    assert table.shape == (0, 8) and not uses.any() and missing.shape == (0,)


def test_tables_and_numbers_that_hold_anything():
    cache = Cache([40, 70, 100], 1, 64, 16, seed=3, spare=9, width=8)         # (entries behind the last page lie outside the pool)
    cache.table[1, 1] = -9
    extremes = [-2**31, 2**31 - 1, -1, 0, 1, 3, 39, 128, 129]
    rng = np.random.default_rng(4)
    for _ in range(12):
        check_fork(cache, uses_of(cache), rng.choice([-2**31, -1, 0, 1, 2, 3, 2**31 - 1], 5), rng.choice(extremes, 5), rng.choice(extremes, 5), layers=1)
    check_fork(cache, rng.choice([-2**31 + 999, -5, 0, 3], cache.pool), [0, 1, 1], [40, 50, 60], [50, 60, 70], layers=1)


def test_large_tables_and_pools():
    rng = np.random.default_rng(5)
    cache = Cache([int(n) for n in rng.integers(1, 9000, 40)], 1, 64, 16, seed=5, spare=5000, width=600)
    cache.table[cache.table >= cache.pool] = -1
    sources = rng.integers(-1, 40, 1100)
    kept = [0 if s < 0 else int(rng.integers(0, cache.lengths[s] + 1)) for s in sources]
    check_fork(cache, uses_of(cache), sources, kept, np.array(kept) + rng.integers(0, 100, 1100), layers=1)


@pytest.mark.parametrize("op", ["compact", "fork", "accept"])
def test_captured_and_replayed(op):
    cache = Cache([60, 45], 2, 64, 16, seed=6, spare=9, width=8)
    cache.table[cache.table >= cache.pool] = -1
    device = cache.device()
    start = [t.clone() for t in device[:4]]
    kept, counts = ints([[0, 2, 5, 11], [1, 2, 4, 7]]), ints([4, 4])
    uses, sources, keep, reserve = ints(uses_of(cache)), ints([0, 0, 1]), ints([40, 37, 45]), ints([50, 50, 50])
    rng = np.random.default_rng(7)
    parents, drafted, sampled = (torch.from_numpy(t).to(DEV) for t in random_drafts(rng, [12, 12], 2))

    def call():
        if op == "compact":
            K.paged_cache_compact_forward([device[:4]], device[4], device[5], kept, counts, 12)
            return device[:4]
        if op == "fork":
            return (*K.paged_cache_fork_forward([device[:4]], device[4], uses, sources, keep, reserve), *device[:4])
        return K.draft_tree_accept_forward(parents, drafted, sampled, device[5])

    def reset():
        for t, s in zip(device[:4], start):
            t.copy_(s)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        kept.copy_(ints([sorted(rng.permutation(12)[:4].tolist()) for _ in range(2)]))
        sources.copy_(ints(rng.integers(-1, 2, 3)))
        keep.copy_(ints(rng.integers(0, 46, 3)))
        sampled.copy_(torch.from_numpy(rng.integers(0, 2, 24)).to(DEV))
        reset()
        want = [t.clone() for t in call()]
        reset()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))


def test_layers_that_share_memory_are_refused():
    cache = Cache([30], 1, 64, 16)
    d = cache.device()
    with pytest.raises(RuntimeError, match="must not share memory"):
        K.paged_cache_compact_forward([d[:4], d[:4]], d[4], d[5], ints([[0, 2]]), ints([2]), 5)
    with pytest.raises(RuntimeError, match="must not share memory"):
        K.paged_cache_fork_forward([d[:4], d[:4]], d[4], ints(uses_of(cache)), ints([0]), ints([5]), ints([9]))
