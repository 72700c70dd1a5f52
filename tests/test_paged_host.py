"""The paged E4M3 operators without a GPU: the index arithmetic that keeps any content of tables, lengths and offsets inside the buffers, the
refusals of the Python functions and of the C entries (nothing is launched), the float64 forms that the GPU tests compare with."""
import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from pocketllm_amd import _ffi, hip_kernel as K

ROOT = Path(__file__).resolve().parents[1]
EXTREMES = [-2**31, -2**31 + 1, -70000, -1, 0, 1, 15, 16, 17, 1000, 2**31 - 2, 2**31 - 1]
needs_library = pytest.mark.skipif(not _ffi.LIB_PATH.exists(), reason="libpllm_hip.so not built")


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    out = tmp_path_factory.mktemp("paged") / "index.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan",
                    str(ROOT / "tests" / "paged_index.cpp"), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    for name in ("first_slot", "slots"):
        getattr(lib, "idx_" + name).restype = ctypes.c_int64
    lib.idx_first_slot.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    lib.idx_slots.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    lib.idx_runs_bound.argtypes = [ctypes.c_int64, ctypes.c_int]
    return lib


def _ints(values):
    return (ctypes.c_int32 * len(values))(*values)


def test_lengths_offsets_and_pages_stay_inside(index):
    for length in EXTREMES:
        for width, shift in ((1, 4), (7, 6), (2**26 - 1, 4), ((2**30 - 1) // 128, 7)):
            assert 0 <= index.idx_length(length, width, shift) <= width << shift
            assert index.idx_length(length, width, shift) == min(max(length, 0), width << shift)
    for rows in (1, 5, 4194303):
        for value in EXTREMES:
            got = index.idx_offset(_ints([value, value, value]), 1, 0, rows)
            assert got == min(max(value, 0), rows) and index.idx_offset(_ints([value, value]), 0, 0, rows) == 0
    assert [index.idx_offset(None, s, 3, 12) for s in range(6)] == [0, 3, 6, 9, 12, 12]
    for pool in (1, 9, 2**31 - 1):
        for entry in EXTREMES:
            row = _ints([entry] * 4)
            for position in EXTREMES:
                page = index.idx_page(row, position, 4, 4, pool)
                assert page == (entry if 0 <= entry < pool and 0 <= position < 64 else -1)


def test_slots_give_every_sequence_its_units(index):
    """The slots of a batch: every unit of every sequence (pages that its new tokens touch; tiles of its rows) has one of its own, inside the grid."""
    rng = random.Random(0)
    for _ in range(400):
        seqs, unit = rng.randint(1, 70), rng.choice([16, 32, 64, 128])
        steps = [rng.choice([0, 1, 2, unit - 1, unit, unit + 1, rng.randint(0, 5 * unit)]) for _ in range(seqs)]
        offsets = np.concatenate([[0], np.cumsum(steps)])
        rows = int(offsets[-1]) + rng.choice([0, 0, 3, 2 * unit])
        for spare, units in ((2, lambda n, at: (at + n - 1) // unit - at // unit + 1 if n else 0), (1, lambda n, at: -(-n // unit))):
            seen, most = set(), index.idx_slots(rows, seqs, unit, spare)
            for s in range(seqs):
                first = index.idx_first_slot(int(offsets[s]), s, unit, spare)
                for i in range(units(steps[s], rng.randint(0, unit - 1))):
                    # the owner that the kernels find: the last sequence whose first slot is not behind it
                    owner = max(c for c in range(seqs) if index.idx_first_slot(int(offsets[c]), c, unit, spare) <= first + i)
                    assert owner == s and first + i < most and first + i not in seen
                    seen.add(first + i)


def test_runs_cover_a_sequence_and_stay_below_their_bound(index):
    for kv_heads in (1, 2, 3, 8, 32, 64, 600, 1024):
        bound = 0
        for length in sorted({1, 2, 255, 256, 257, 511, 512, 4096, 16383, 16384, 16385, 100001, 131072, 10**6, 2**30 - 1} | {random.Random(kv_heads).randint(1, 300000) for _ in range(300)}):
            keys, runs = index.idx_run_keys(length, kv_heads), index.idx_runs(length, kv_heads)
            assert keys % 256 == 0 and (runs - 1) * keys < length <= runs * keys
            assert runs <= index.idx_runs_bound(length, kv_heads)
            assert index.idx_runs_bound(length, kv_heads) >= bound                # a longer table has room for the runs of every shorter sequence
            bound = index.idx_runs_bound(length, kv_heads)
        assert index.idx_runs(0, kv_heads) == 0 and [index.idx_runs_bound(n, kv_heads) for n in (0, 1, 1024)] == [1, 1, 1]
        assert index.idx_runs(1024, kv_heads) == 1 and index.idx_runs(1025, kv_heads) == 3


def test_pages_that_a_number_of_tokens_touches(index):
    index.idx_pages_touched.restype = ctypes.c_int64
    for page in (16, 32, 64, 128):
        for steps in list(range(1, 300)) + [4096, 2**31]:
            assert index.idx_pages_touched(ctypes.c_int64(steps), ctypes.c_int64(page)) == max((at + steps - 1) // page + 1 for at in range(page))


def test_blocks_that_see_so_many_tiles(index):
    """The closed form by which the prompt kernel orders its blocks against a count."""
    rng = random.Random(1)
    for _ in range(300):
        group, block, n = rng.choice([1, 3, 6, 8]), rng.choice([128, 256]), rng.choice([0, 1, rng.randint(1, 300)])
        keys = n + rng.choice([0, -n, rng.randint(-n, 0), rng.randint(0, 1000)])
        rows = n * group
        blocks = [min(rows, block * (b + 1)) - 1 for b in range(-(-rows // block))]      # their last rows
        sees = [max(0, keys - n + r // group + 1) for r in blocks]
        for tiles in range(0, 25):
            want = sum(tiles == 0 or -(-v // 64) >= tiles for v in sees)
            assert index.idx_blocks_seeing(tiles, rows, keys - n, group, block) == want, (tiles, rows, keys, n, group, block)


def test_e4m3_of_the_oracle_is_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), P.e4m3_values(), equal_nan=True)
    v = torch.cat([torch.randn(5000, generator=torch.Generator().manual_seed(0)) * 10.0 ** k for k in range(-4, 3)]).clamp(-448, 448)
    assert np.array_equal(v.to(torch.float8_e4m3fn).double().numpy(), P.e4m3_round(v.double().numpy()))
    for amax in (1.0, 447.9, 448.0, 448.0001, 1e-30, 3e38, 0.0):
        s = float(P.page_scale(amax))
        assert amax / s <= 448 and (amax / s > 224 or s == 2.0 ** -120)


def _cache(seqs=2, pool=4, kv_heads=2, page=16, dim=64, width=3):
    f8 = torch.float8_e4m3fn
    return dict(key_pages=torch.zeros(pool, kv_heads, page, dim, dtype=torch.uint8).view(f8), value_pages=torch.zeros(pool, kv_heads, dim, page, dtype=torch.uint8).view(f8),
                key_scales=torch.ones(pool, kv_heads), value_scales=torch.ones(pool, kv_heads), block_table=torch.zeros(seqs, width, dtype=torch.int32),
                lengths=torch.ones(seqs, dtype=torch.int32))


BAD_CACHE = [
    (dict(key_pages=torch.zeros(4, 2, 16 * 64, dtype=torch.uint8)), "pages must be"), (dict(value_pages=torch.zeros(4, 2, 16, 64, dtype=torch.uint8)), "pages must be"),
    (dict(key_pages=torch.zeros(4, 2, 16, 64)), "float8_e4m3fn"), (dict(value_pages=torch.zeros(4, 2, 64, 16, dtype=torch.float16)), "float8_e4m3fn"),
    (dict(key_scales=torch.ones(4, 2, dtype=torch.float16)), "scales must be"), (dict(value_scales=torch.ones(4, 1)), "scales must be"),
    (dict(value_scales=torch.ones(2, 4).t()), "scales must be"), (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), "block_table"), (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()), "block_table"),
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), "block_table"),
    (dict(lengths=torch.ones(2)), "lengths"), (dict(lengths=torch.ones(3, dtype=torch.int32)), "lengths"), (dict(), "one CUDA device"),
]


@pytest.mark.parametrize("bad,words", BAD_CACHE)
def test_caches_are_refused(bad, words):
    cache = {**_cache(), **bad}
    q, k, cu = torch.zeros(2, 4 * 64, dtype=torch.bfloat16), torch.zeros(2, 2 * 64, dtype=torch.bfloat16), torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match=words):
        K.paged_attention_decode_forward(q, **cache)
    with pytest.raises(RuntimeError, match=words):
        K.paged_attention_prompt_forward(q, **cache, cu_steps=cu)
    with pytest.raises(RuntimeError, match=words):
        K.paged_kv_append_forward(q, k, k, **cache)


@pytest.mark.parametrize("page,dim", [(8, 64), (24, 64), (256, 64), (16, 80), (16, 256)])
def test_page_and_head_sizes_are_refused(page, dim):
    for scale in (-1.0, float("nan"), float("inf"), 3e38):
        with pytest.raises(RuntimeError, match="scale must be" if page == 16 and dim == 64 else "pages of 16"):
            K.paged_attention_decode_forward(torch.zeros(2, 4 * dim, dtype=torch.float16), **_cache(page=page, dim=dim), scale=scale)
    with pytest.raises(RuntimeError, match="pages of 16"):
        K.paged_attention_decode_forward(torch.zeros(2, 4 * dim, dtype=torch.float16), **_cache(page=page, dim=dim))


def test_types_are_refused():
    for dtype in (torch.float32, torch.float64, torch.int16):
        q = torch.zeros(2, 256).to(dtype)
        with pytest.raises(RuntimeError, match="float16 or bfloat16"):
            K.paged_attention_decode_forward(q, **_cache())
        with pytest.raises(RuntimeError, match="float16 or bfloat16"):
            K.paged_kv_append_forward(None, q[:, :128], q[:, :128], **_cache())


BAD_NORM = [
    (dict(x=torch.zeros(2, 100)), "multiple of 128"), (dict(x=torch.zeros(2, 32896)), "multiple of 128"), (dict(x=torch.zeros(2, 256, dtype=torch.float64)), "x must be"),
    (dict(weight=torch.ones(255)), "weight must be"), (dict(weight=torch.ones(256, dtype=torch.bfloat16)), "weight must be"), (dict(), "one CUDA device"),
]


@pytest.mark.parametrize("bad,words", BAD_NORM)
def test_norms_are_refused(bad, words):
    given = {**dict(x=torch.zeros(2, 256), weight=torch.ones(256)), **bad}
    with pytest.raises(RuntimeError, match=words):
        K.fused_add_rms_norm_fp8_forward(given["x"], None, given["weight"], 1e-6)


@needs_library
def test_c_entries_refuse_before_anything_is_launched():
    """Addresses that no kernel may see: every call here ends in a status."""
    lib = _ffi.load_library()
    at = 4096
    base = dict(q=at, q_stride=256, dtype=1, kp=at, vp=at, ks=at, vs=at, pool=4, page=16, table=at, table_stride=3, width=3, lengths=at)

    def decode(**kw):
        a = {**base, **dict(seqs=2, steps=1, heads=4, kv=2, dim=64, scale=0.1, out=at, ws=None, need=0), **kw}
        return lib.pllm_paged_attention_decode(*a.values(), None)

    def prompt(**kw):
        a = {**base, **dict(cu=at, tokens=5, seqs=2, heads=4, kv=2, dim=64, scale=0.1, out=at, ws=None, need=0), **kw}
        return lib.pllm_paged_attention_prompt(*a.values(), None)

    def append(**kw):
        a = {**dict(q=at, q_stride=256, k=at, k_stride=128, v=at, v_stride=128, dtype=1, q_out=at, kp=at, vp=at, ks=at, vs=at, pool=4, page=16, table=at, table_stride=3, width=3,
                    lengths=at, cu=at, cos=at, sin=at, positions=48, rope=64, rows=5, seqs=2, heads=4, kv=2, dim=64), **kw}
        return lib.pllm_paged_kv_append(*a.values(), None)

    invalid, unsupported, workspace = -1, -2, -4
    for call in (decode, prompt):
        for kw in (dict(q=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(table=None), dict(lengths=None), dict(out=None), dict(dtype=0), dict(dtype=3),
                   dict(seqs=0), dict(heads=0), dict(kv=0), dict(heads=3), dict(pool=0), dict(width=0), dict(table_stride=2), dict(q_stride=255), dict(q=at + 2), dict(q_stride=257),
                   dict(kp=at + 8), dict(table=at + 2), dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38)):
            assert call(**kw) == invalid, kw
        for kw in (dict(page=8), dict(page=256), dict(dim=96, q_stride=512), dict(pool=2**31), dict(width=2**28, table_stride=2**28), dict(seqs=10**6), dict(heads=2048, q_stride=2**20)):
            assert call(**kw) == unsupported, kw
    assert decode(steps=0) == invalid and decode(steps=5000) == unsupported and prompt(cu=None) == invalid and prompt(tokens=0) == invalid and prompt(tokens=2**23) == unsupported
    assert decode(width=300, table_stride=300) == workspace
    need = lib.pllm_paged_attention_decode_workspace_bytes(2, 1, 4, 2, 64, 4800)
    assert need >= 2 * 4 * 10 * 66 * 4 and decode(width=300, table_stride=300, ws=at, need=need - 1) == workspace
    assert lib.pllm_paged_attention_decode_workspace_bytes(2, 1, 4, 2, 64, 1024) == 0 and lib.pllm_paged_attention_decode_workspace_bytes(-1, 1, 4, 2, 64, 256) == 0
    assert prompt(width=200, table_stride=200) == workspace
    need = lib.pllm_paged_attention_prompt_workspace_bytes(5, 2, 4, 2, 64, 3200)
    assert need >= 2 * 10 * 2 * 7 * 66 * 4 and prompt(width=200, table_stride=200, ws=at, need=need - 1) == workspace
    assert lib.pllm_paged_attention_prompt_workspace_bytes(5, 2, 4, 2, 64, 511) == 0 and lib.pllm_paged_attention_prompt_workspace_bytes(100000, 1, 4, 2, 64, 10**6) == 0
    # what sequences of few rows keep between two launches stays below a gigabyte, whatever the batch
    for seqs, kv, positions in ((1, 8, 10**6), (64, 8, 131072), (2000, 8, 131072), (65535, 1, 10**6), (300, 64, 40000)):
        assert lib.pllm_paged_attention_prompt_workspace_bytes(100000, seqs, 2 * kv, kv, 128, positions) <= 2**30 + 512
    for kw in (dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(dtype=0), dict(rows=0), dict(seqs=0), dict(kv=0), dict(heads=0), dict(pool=0), dict(width=0),
               dict(table_stride=1), dict(cu=None), dict(k_stride=127), dict(v_stride=120), dict(q_stride=200), dict(rope=-16), dict(rope=80), dict(cos=None), dict(sin=None),
               dict(positions=47), dict(k=at + 8), dict(cos=at + 4), dict(k_stride=132), dict(lengths=at + 1)):
        assert append(**kw) == invalid, kw
    for kw in (dict(rope=8), dict(page=48, positions=999), dict(dim=32, rope=16), dict(rows=2**23), dict(seqs=2**21), dict(kv=2000, k_stride=2**18, v_stride=2**18), dict(pool=2**32),
               dict(rows=2**21, kv=512, k_stride=2**16, v_stride=2**16)):
        assert append(**kw) == unsupported, kw

    def norm(**kw):
        a = {**dict(x=at, r=at, dtype=1, w=at, total=at, codes=at, scales=at, rows=2, dim=256, eps=1e-6, qe=1e-4, pow2=0), **kw}
        return lib.pllm_fused_add_rms_norm_fp8(*a.values(), None)

    for kw in (dict(x=None), dict(w=None), dict(total=None), dict(codes=None), dict(scales=None), dict(dtype=3), dict(rows=0), dict(dim=0), dict(dim=100), dict(x=at + 2), dict(r=at + 8),
               dict(codes=at + 4), dict(scales=at + 2), dict(qe=0.0), dict(qe=float("nan"))):
        assert norm(**kw) == invalid, kw
    assert norm(dim=32896) == unsupported and norm(rows=2**23) == unsupported
