"""Serving by drafted trees without a GPU: the index arithmetic of trees, the refusals of the Python functions and of the C entries (nothing is launched), the float64
forms that the GPU tests compare with."""
import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import tree_oracle as T
from pocketllm_amd import _ffi, hip_kernel as K
from test_paged_host import BAD_CACHE, _cache

ROOT = Path(__file__).resolve().parents[1]
EXTREMES = [-2**31, -2**31 + 1, -70000, -257, -1, 0, 1, 63, 64, 255, 256, 2**31 - 1]
needs_library = pytest.mark.skipif(not _ffi.LIB_PATH.exists(), reason="libpllm_hip.so not built")


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    out = tmp_path_factory.mktemp("tree") / "index.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan",
                    str(ROOT / "tests" / "tree_index.cpp"), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.idx_tree_window.restype = ctypes.c_uint64
    lib.idx_tree_window.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64]
    return lib


def _bits(index, parents, i, words=4):
    got = (ctypes.c_uint64 * words)()
    (index.idx_tree_ancestors if words == 4 else index.idx_tree_ancestors_one)((ctypes.c_int32 * len(parents))(*parents), i, got)
    return sum(int(w) << (64 * k) for k, w in enumerate(got))


def test_ancestors_end_whatever_the_parents_are(index):
    rng = random.Random(0)
    for n in (1, 2, 63, 64, 65, 200, 256):
        for parents in ([-1] + [rng.randint(-1, i - 1) for i in range(1, n)], list(range(-1, n - 1)), [rng.choice(EXTREMES) for _ in range(n)], [(i + 1) % n for i in range(n)]):
            family = T.ancestors(parents)
            for i in {0, n // 2, n - 1}:
                want = sum(1 << k for k in range(n) if family[i, k])
                assert _bits(index, parents, i) == want
                if n <= 64:
                    assert _bits(index, parents, i, 1) == want
    assert _bits(index, [-1] * 256, 256) == 0                                 # (a node behind the last one that a tree can have)


def test_windows_are_what_a_node_sees(index):
    rng = random.Random(1)
    for _ in range(4000):
        words = rng.choice([1, 4])
        mask = rng.getrandbits(64 * words)
        bits = (ctypes.c_uint64 * words)(*[mask >> (64 * w) & (2**64 - 1) for w in range(words)])
        past = rng.choice([rng.randint(-300, 700), -512, 2**30 - 5])
        first = max(0, past + rng.randint(-130, 64 * words + 70))
        limit = rng.choice([past + rng.randint(0, 300), 0, 2**30 - 1, first + rng.randint(0, 70)])
        want = sum(1 << i for i in range(64) if first + i < limit and (first + i < past or (first + i - past < 64 * words and mask >> (first + i - past) & 1)))
        assert index.idx_tree_window(bits, words, past, first, limit) == want


def test_pasts_stay_in_range(index):
    for length in EXTREMES:
        for n in (0, 1, 64, 256, 4194303):
            assert index.idx_tree_past(length, n) == max(length - n, -512)


def _trees(tokens=2):
    return dict(parents=torch.full((tokens,), -1, dtype=torch.int32))


@pytest.mark.parametrize("bad,words", BAD_CACHE)
def test_caches_are_refused(bad, words):
    cache = {**_cache(), **bad}
    q, cu = torch.zeros(2, 4 * 64, dtype=torch.bfloat16), torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match=words):
        K.paged_attention_tree_forward(q, **cache, **_trees(), cu_steps=cu)


def _layers(count=2, **kw):
    caches = [_cache(**kw) for _ in range(count)]
    return [(c["key_pages"], c["value_pages"], c["key_scales"], c["value_scales"]) for c in caches], caches[0]["block_table"], caches[0]["lengths"]


BAD_TREES = [
    (dict(q=torch.zeros(2, 1, 256, dtype=torch.bfloat16)), "q must be"), (dict(q=torch.zeros(2, 250, dtype=torch.bfloat16)), "one CUDA device|heads must be"),
    (dict(parents=torch.zeros(2, dtype=torch.int64)), "one CUDA device|parents"), (dict(cu_steps=torch.zeros(2, dtype=torch.int32)), "one CUDA device|cu_steps"),
    (dict(scale=-1.0), "one CUDA device|scale"), (dict(q=torch.zeros(2, 256)), "float16 or bfloat16"),
]


@pytest.mark.parametrize("bad,words", BAD_TREES)
def test_trees_are_refused(bad, words):
    given = {**dict(q=torch.zeros(2, 256, dtype=torch.bfloat16), **_trees()), **bad}
    with pytest.raises(RuntimeError, match=words):
        K.paged_attention_tree_forward(**given, **_cache())


BAD_SAMPLES = [
    (dict(logits=torch.zeros(8)), "logits must be"), (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), "logits must be"), (dict(logits=torch.zeros(2, 0)), "vocabulary"),
    (dict(logits=torch.zeros(1, 2**20 + 1), uniform=torch.zeros(1)), "vocabulary"), (dict(logits=torch.zeros(65536, 2), uniform=torch.zeros(65536)), "rows"),
    (dict(uniform=torch.zeros(3)), "uniform"), (dict(uniform=torch.zeros(2, dtype=torch.float64)), "uniform"), (dict(uniform=torch.zeros(4)[::2]), "uniform"),
    (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=torch.ones(2, dtype=torch.float64)), "temperature"),
    (dict(temperature=torch.ones(3)), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_k=2.5), "top_k"), (dict(top_k=torch.ones(2)), "top_k"),
    (dict(top_p=-0.1), "top_p"), (dict(top_p=torch.ones(2, dtype=torch.float16)), "top_p"), (dict(min_p=1.5), "min_p"), (dict(min_p=-0.1), "min_p"), (dict(), "one CUDA device"),
]


@pytest.mark.parametrize("bad,words", BAD_SAMPLES)
def test_samples_are_refused(bad, words):
    given = {**dict(logits=torch.zeros(2, 8), uniform=torch.zeros(2)), **bad}
    with pytest.raises(RuntimeError, match=words):
        K.sample_tokens_forward(**given)


BAD_PATHS = [
    (dict(parents=torch.zeros(4)), "parents"), (dict(drafted=torch.zeros(4, dtype=torch.int32)), "drafted"), (dict(sampled=torch.zeros(3, dtype=torch.int64)), "sampled"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), "same number"), (dict(most=0), "most"), (dict(most=257), "most"),
    (dict(cu_steps=torch.zeros(2, dtype=torch.int32)), "cu_steps"), (dict(), "one CUDA device"),
    (dict(parents=torch.zeros(514, dtype=torch.int32), drafted=torch.zeros(514, dtype=torch.int64), sampled=torch.zeros(514, dtype=torch.int64)), "at most 256"),
]


@pytest.mark.parametrize("bad,words", BAD_PATHS)
def test_paths_are_refused(bad, words):
    given = {**dict(parents=torch.zeros(4, dtype=torch.int32), drafted=torch.zeros(4, dtype=torch.int64), sampled=torch.zeros(4, dtype=torch.int64),
                    lengths=torch.ones(2, dtype=torch.int32)), **bad}
    with pytest.raises(RuntimeError, match=words):
        K.draft_tree_accept_forward(**given)


def test_page_operators_refuse():
    layers, table, lengths = _layers()
    kept, counts, rows = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="one CUDA device"):
        K.paged_cache_compact_forward(layers, table, lengths, kept, counts, 3)
    with pytest.raises(RuntimeError, match="one CUDA device"):
        K.paged_cache_fork_forward(layers, table, torch.zeros(4, dtype=torch.int32), rows, rows, rows)
    for bad in ([], [layers[0][:3]]):
        with pytest.raises(RuntimeError, match="layers must be"):
            K.paged_cache_compact_forward(bad, table, lengths, kept, counts, 3)
        with pytest.raises(RuntimeError, match="layers must be"):
            K.paged_cache_fork_forward(bad, table, torch.zeros(4, dtype=torch.int32), rows, rows, rows)


@needs_library
def test_c_entries_refuse_before_anything_is_launched():
    """Addresses that no kernel may see: every call here ends in a status."""
    lib, at = _ffi.load_library(), 4096
    invalid, unsupported, workspace = -1, -2, -4

    def tree(**kw):
        a = {**dict(q=at, q_stride=256, dtype=1, kp=at, vp=at, ks=at, vs=at, pool=4, page=16, table=at, table_stride=3, width=3, lengths=at, parents=at, cu=at, tokens=6, seqs=2,
                    heads=4, kv=2, dim=64, scale=0.1, out=at, ws=None, need=0), **kw}
        return lib.pllm_paged_attention_tree(*a.values(), None)

    for kw in (dict(q=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(table=None), dict(lengths=None), dict(parents=None), dict(out=None), dict(dtype=0),
               dict(tokens=0), dict(seqs=0), dict(heads=3), dict(kv=0), dict(pool=0), dict(width=0), dict(table_stride=2), dict(q_stride=255), dict(q=at + 2), dict(parents=at + 2),
               dict(cu=None, tokens=5), dict(scale=float("nan"))):
        assert tree(**kw) == invalid, kw
    for kw in (dict(page=8), dict(dim=96, q_stride=512), dict(pool=2**31), dict(width=2**28, table_stride=2**28), dict(seqs=10**6), dict(cu=None, tokens=514), dict(tokens=2**23)):
        assert tree(**kw) == unsupported, kw
    for even in (0, 1):
        need = lib.pllm_paged_attention_tree_workspace_bytes(6, 2, even, 4, 2, 64, 3200)
        assert need > 0 and tree(cu=None if even else at, width=200, table_stride=200, ws=at, need=need - 1) == workspace
    assert lib.pllm_paged_attention_tree_workspace_bytes(0, 2, 1, 4, 2, 64, 3200) == 0

    def append(**kw):
        a = {**dict(q=at, q_stride=256, k=at, k_stride=128, v=at, v_stride=128, dtype=1, q_out=at, kp=at, vp=at, ks=at, vs=at, pool=4, page=16, table=at, table_stride=3, width=3,
                    lengths=at, cu=at, cos=at, sin=at, positions=4, at=at, rope=64, rows=5, seqs=2, heads=4, kv=2, dim=64), **kw}
        return lib.pllm_paged_kv_append_at(*a.values(), None)

    for kw in (dict(at=None), dict(positions=0), dict(at=at + 1), dict(cos=None)):
        assert append(**kw) == invalid, kw

    def accept(**kw):
        a = {**dict(parents=at, drafted=at, sampled=at, lengths=at, cu=at, rows=6, seqs=2, most=8, kept=at, counts=at, tokens=at, news=at), **kw}
        return lib.pllm_draft_tree_accept(*a.values(), None)

    for kw in (dict(parents=None), dict(drafted=None), dict(sampled=None), dict(lengths=None), dict(kept=None), dict(counts=None), dict(tokens=None), dict(news=None), dict(rows=0),
               dict(seqs=0), dict(most=0), dict(cu=None, rows=5), dict(drafted=at + 4), dict(parents=at + 2)):
        assert accept(**kw) == invalid, kw
    for kw in (dict(most=257), dict(rows=2**23), dict(seqs=2**21), dict(cu=None, rows=514)):
        assert accept(**kw) == unsupported, kw

    far = 1 << 40
    caches = lambda *addresses: (ctypes.c_void_p * len(addresses))(*addresses)
    good = caches(*[far + (i << 30) for i in range(8)])

    def compact(**kw):
        a = {**dict(caches=good, layers=2, pool=4, page=16, table=at, table_stride=3, width=3, lengths=at, kept=at, most=8, counts=at, cu=at, steps=0, seqs=2, kv=2, dim=64), **kw}
        return lib.pllm_paged_cache_compact(*a.values(), None)

    def fork(**kw):
        a = {**dict(caches=good, layers=2, pool=4, page=16, table=at, table_stride=3, width=3, uses=at, sources=at, kept=at, reserve=at, seqs=2, rows=2, kv=2, dim=64, new_table=at,
                    new_uses=at, missing=at, ws=at, need=10**6), **kw}
        return lib.pllm_paged_cache_fork(*a.values(), None)

    twice = caches(*[far + (i % 4 << 30) for i in range(8)])
    near = caches(far, far + 8192, far + (1 << 30), far + (2 << 30))              # the second layer's half of a pool away
    for call in (compact, fork):
        for kw in (dict(caches=None), dict(layers=0), dict(pool=0), dict(width=0), dict(table=None), dict(table_stride=2), dict(kept=None), dict(seqs=0), dict(kv=0),
                   dict(caches=caches(0, far, far, far), layers=1), dict(caches=caches(far + 8, far + (1 << 30), far + (2 << 30), far + (3 << 30)), layers=1),
                   dict(caches=twice), dict(caches=near, layers=1, pool=5), dict(table=at + 2)):
            assert call(**kw) == invalid, kw
        for kw in (dict(page=8), dict(dim=96), dict(pool=2**31), dict(width=2**28, table_stride=2**28), dict(seqs=10**6), dict(kv=2000), dict(layers=1025)):
            assert call(**kw) == unsupported, kw
    assert compact(lengths=None) == invalid and compact(counts=None) == invalid and compact(cu=None) == invalid and compact(most=0) == invalid
    assert compact(most=257) == unsupported and compact(cu=None, steps=257) == unsupported
    for name in ("uses", "sources", "reserve", "new_table", "new_uses", "missing"):
        assert fork(**{name: None}) == invalid
    assert fork(rows=0) == invalid and fork(rows=65535) == unsupported
    assert fork(rows=60000, width=40000, table_stride=40000) == unsupported      # (more pages than 32 bits count)
    assert fork(need=lib.pllm_paged_cache_fork_workspace_bytes(2, 4) - 1) == workspace and fork(ws=None) == workspace

    def sample(**kw):
        a = {**dict(logits=at, stride=100, dtype=1, uniform=at, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0, m=None, m_all=0.0, rows=2, vocab=100, tokens=at, ws=at,
                    need=10**8), **kw}
        return lib.pllm_sample_tokens(*a.values(), None)

    for kw in (dict(logits=None), dict(uniform=None), dict(tokens=None), dict(rows=0), dict(vocab=0), dict(stride=99), dict(dtype=3), dict(dtype=-1), dict(logits=at + 1),
               dict(dtype=0, logits=at + 2), dict(uniform=at + 2), dict(tokens=at + 4), dict(ws=at + 8), dict(t_all=-1.0), dict(t_all=float("nan")), dict(k_all=-1), dict(p_all=-0.5),
               dict(m_all=1.5), dict(k=at + 1)):
        assert sample(**kw) == invalid, kw
    assert sample(rows=65536) == unsupported and sample(vocab=2**20 + 1, stride=2**21) == unsupported
    assert sample(need=lib.pllm_sample_tokens_workspace_bytes(2, 100, 1) - 1) == workspace and sample(ws=None) == workspace
    assert lib.pllm_sample_tokens_workspace_bytes(0, 100, 1) == 0


def test_oracle_of_samples():
    x = [1.0, 3.0, 3.0, float("nan"), -np.inf, 2.0]
    assert T.sample(x, 0.9, temperature=0.0)[0] == 1 and T.sample([np.nan, -np.inf], 0.5)[0] == -1
    # equal weights: the cuts by index
    assert [T.sample([0.0] * 4, u)[0] for u in (0.0, 0.25, 0.5, 0.999, 1.0)] == [0, 1, 2, 3, 3]
    assert [T.sample([0.0] * 4, u, top_k=2)[0] for u in (0.0, 0.5, 0.999)] == [0, 1, 1]
    assert [T.sample([0.0] * 4, u, top_p=0.5)[0] for u in (0.0, 0.5, 0.999)] == [0, 1, 1]
    assert T.sample([0.0, 1.0, 0.9], 0.0, min_p=0.8)[0] == 1 and T.sample([np.inf, 5.0, np.inf], 0.9)[0] == 2
    rng = np.random.default_rng(0)
    x = rng.standard_normal(50)
    share = np.exp(x - x.max())
    share[np.argsort(-x)[9:]] = 0
    got = np.bincount([T.sample(x, u, top_k=9)[0] for u in (np.arange(4000) + 0.5) / 4000], minlength=50) / 4000
    assert np.abs(got - share / share.sum()).max() <= 1 / 4000


def test_oracle_of_forks():
    table = np.array([[3, 4, 5], [0, 1, -1]])
    uses = np.array([1, 1, 0, 1, 1, 1, 0, 0])
    # two rows out of the first (8 of 12 tokens: whole pages; 10: one in part), the second ends
    out, after, missing, copies = T.fork(table, uses, [0, 0, 0], [8, 10, 11], [9, 10, 13], 4)
    assert out.tolist() == [[3, 4, 0], [3, 4, 5], [3, 4, 1]] and copies == [(5, 1)] and missing.tolist() == [0, 0, 0]    # (width * page bounds the third)
    assert after.tolist() == [1, 1, 0, 3, 3, 1, 0, 0]
    out, after, missing, copies = T.fork(table, uses + np.array([0, 0, 0, 0, 0, 1, 0, 0]), [0, -1], [10, 5], [12, 12], 4)
    assert out.tolist() == [[3, 4, 0], [1, 2, 6]] and copies == [(5, 0)] and after.tolist() == [1, 1, 1, 1, 1, 1, 1, 0]
