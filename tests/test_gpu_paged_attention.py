"""Attention over the paged E4M3 cache (decode and prompt forms) against a float64 form, where it can go wrong: lengths of none and one, ends inside
pages and tiles, heads that do not fill tiles, pages that are missing, NaN behind the last key and in keys that a query does not see."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from pocketllm_amd import _ffi, hip_kernel as K
from paged_cases import DEV, Cache, close, queries

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _even(seqs, steps):
    return np.arange(seqs + 1) * steps


def _decode(cache, q, **kw):
    return K.paged_attention_decode_forward(q.to(DEV), *cache.device(), **kw)


# (lengths, steps, heads, kv_heads, dim, page, dtype)
DECODE = [
    ([1], 1, 1, 1, 64, 16, BF), ([1, 2, 15, 16, 17], 1, 6, 1, 128, 16, HF), ([31, 32, 33, 63, 64, 65], 1, 8, 2, 128, 32, BF),
    ([0, 255, 256, 257, 0, 300], 1, 12, 2, 128, 64, BF), ([700, 1, 513], 1, 32, 32, 64, 16, HF), ([1025, 130], 1, 48, 8, 128, 128, HF),
    ([4, 3, 2, 1, 0, 260], 4, 6, 1, 128, 64, BF), ([77, 640, 1000], 3, 40, 8, 64, 32, HF), ([515, 64], 5, 16, 1, 128, 16, BF), ([2000], 2, 48, 8, 128, 64, HF),
    ([9, 4100], 1, 5, 1, 128, 128, BF), ([129, 258], 17, 2, 2, 64, 64, BF),
]


@pytest.mark.parametrize("lengths,steps,heads,kv_heads,dim,page,dtype", DECODE)
def test_decode_against_float64(lengths, steps, heads, kv_heads, dim, page, dtype):
    cache = Cache(lengths, kv_heads, dim, page, seed=sum(lengths) + heads)
    q = queries(len(lengths) * steps, heads, dim, dtype, seed=steps)
    got = _decode(cache, q.view(len(lengths), steps, -1))
    assert got.dtype == dtype and got.shape == (len(lengths), steps, heads * dim)
    close(got, *cache.attention(q.view(-1, heads, dim).double().numpy(), _even(len(lengths), steps)), dtype)


# (steps, pasts, heads, kv_heads, dim, page, dtype)
PROMPT = [
    ([1], [0], 1, 1, 64, 16, BF), ([5, 0, 17], [0, 3, 40], 6, 1, 128, 16, HF), ([33, 1, 64], [31, 100, 0], 8, 2, 128, 32, BF),
    ([130, 65], [0, 63], 4, 4, 64, 64, HF), ([20, 129, 3], [500, 0, 62], 12, 2, 128, 128, BF), ([257], [0], 5, 1, 128, 64, BF), ([40, 40], [24, 0], 48, 8, 128, 64, HF),
    ([300], [77], 2, 2, 64, 16, BF),
]


@pytest.mark.parametrize("steps,pasts,heads,kv_heads,dim,page,dtype", PROMPT)
def test_prompt_against_float64(steps, pasts, heads, kv_heads, dim, page, dtype):
    cache = Cache([n + p if n else 0 for n, p in zip(steps, pasts)], kv_heads, dim, page, seed=sum(steps) + heads)
    cu = np.concatenate([[0], np.cumsum(steps)])
    q = queries(cu[-1], heads, dim, dtype, seed=1)
    got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
    assert got.dtype == dtype and got.shape == q.shape
    close(got, *cache.attention(q.view(-1, heads, dim).double().numpy(), cu), dtype)


def test_rows_behind_the_last_sequence_and_sequences_without_keys_are_zeros():
    cache = Cache([40, 0, 10], 2, 128, 16, seed=5)
    cu = np.array([0, 30, 34, 40])                                            # the second has four tokens and no position for them
    q = queries(200, 6, 128, BF)
    got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
    want, note = cache.attention(q[:40].view(-1, 6, 128).double().numpy(), cu)
    close(got[:40], want, note, BF)
    assert (got[30:34] == 0).all() and (got[40:] == 0).all()


@pytest.mark.parametrize("form", ["decode", "prompt"])
def test_missing_pages_hold_no_keys(form):
    """Table entries outside the pool in the middle of a sequence: their keys have no weight; a sequence of nothing else has zeros."""
    cache = Cache([200, 64, 100], 2, 128, 32, seed=7)
    cache.table[0, 2], cache.table[0, 4] = -1, cache.pool
    cache.table[1, :] = np.iinfo(np.int32).min
    cache.table[2, 0] = np.iinfo(np.int32).max
    q = queries(3, 4, 128, BF)
    if form == "decode":
        got = _decode(cache, q)
    else:
        got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.arange(4, dtype=torch.int32, device=DEV))
    close(got, *cache.attention(q.view(-1, 4, 128).double().numpy(), _even(3, 1)), BF)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("form", ["decode", "prompt"])
def test_lengths_that_the_table_does_not_hold(form):
    """Lengths beyond the table end with it, negative ones are none."""
    cache = Cache([96, 96, 5], 1, 64, 16, seed=8)
    cache.lengths[:] = [97 + 300, -4, 5]
    q = queries(3, 2, 64, HF)
    if form == "decode":
        got = _decode(cache, q)
    else:
        got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.arange(4, dtype=torch.int32, device=DEV))
    close(got, *cache.attention(q.view(-1, 2, 64).double().numpy(), _even(3, 1)), HF)


@pytest.mark.parametrize("form", ["decode", "prompt"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_nan_and_infinite_values_reach_only_the_queries_that_see_them(form, dtype):
    """The last of three new tokens has NaN values and a NaN key: the two queries before it do not see either; an older NaN value reaches all
    queries in its own dimension."""
    cache = Cache([70, 131], 1, 128, 64, seed=9)
    page, slot = cache.table[0, 69 // 64], 69 % 64
    cache.value_codes[page, 0, 3:9, slot] = 0x7f
    page, slot = cache.table[1, 130 // 64], 130 % 64
    cache.key_codes[page, 0, slot, 17] = 0xff
    cache.value_codes[cache.table[1, 0], 0, 100, 5] = 0xff
    q = queries(6, 6, 128, dtype)
    if form == "decode":
        got = _decode(cache, q.view(2, 3, -1))
    else:
        got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV))
    want, note = cache.attention(q.view(-1, 6, 128).double().numpy(), _even(2, 3))
    assert np.isnan(want[2, :, 3:9]).all() and not np.isnan(want[:2]).any() and np.isnan(want[5]).all() and np.isnan(want[3:5, :, 100]).all()
    close(got, want, note, dtype)


@pytest.mark.parametrize("form", ["decode", "prompt"])
def test_scores_past_the_exponent_and_scales_far_apart(form):
    """Scores of thousands, pages whose scales differ by 2^30 and more, values at the top of fp16, huge bf16 queries against tiny keys."""
    for dtype, size, exponents in ((BF, 30.0, (-30, 4)), (HF, 40.0, (-16, 3)), (BF, 1e30, (-118, -100))):
        cache = Cache([150, 90], 1, 128, 16, seed=10, scale_exponents=exponents)
        if dtype == HF:
            cache.value_scales[cache.table[0, 1]] = 2.0 ** 8
            cache.value_codes[cache.table[0, 1]] = 0x78                        # 256 * 2^8 = 65536, what fp16's largest values round up to
        q = queries(2, 3, 128, dtype, size=size)
        if form == "decode":
            got = _decode(cache, q)
        else:
            got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV))
        want, note = cache.attention(q.view(-1, 3, 128).double().numpy(), _even(2, 1))
        top = torch.finfo(dtype).max
        keep = np.abs(want) < top * 0.98                                       # (outputs beyond the type are infinities)
        close(torch.where(torch.from_numpy(keep.reshape(got.shape)).to(DEV), got, torch.zeros_like(got)), np.where(keep, want, 0.0), note, dtype)


def test_scale_strides_and_narrow_tables():
    cache = Cache([100, 37], 2, 128, 16, seed=11, width=20)
    heads = 6
    q = queries(2, heads, 128, BF)
    kp, vp, ks, vs, table, lengths = cache.device()
    want = K.paged_attention_decode_forward(q.to(DEV), kp, vp, ks, vs, table, lengths, scale=0.3)
    close(want, *cache.attention(q.view(-1, heads, 128).double().numpy(), _even(2, 1), scale=0.3), BF)
    # the queries as columns of a fused projection, at an odd place too; a table that is part of a wider one; codes as bytes
    wide = torch.randn(2, heads * 128 + 512, device=DEV).to(BF)
    wide[:, 256:256 + heads * 128] = q.to(DEV)
    odd = torch.randn(2, heads * 128 + 3, device=DEV).to(BF)
    odd[:, 3:] = q.to(DEV)
    for view in (wide[:, 256:256 + heads * 128], odd[:, 3:]):
        for t in (table, table[:, :7]):
            assert torch.equal(K.paged_attention_decode_forward(view, kp.view(torch.uint8), vp.view(torch.uint8), ks, vs, t, lengths, scale=0.3), want)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    a = K.paged_attention_prompt_forward(q.to(DEV), kp, vp, ks, vs, table, lengths, cu, scale=0.3)
    assert torch.equal(K.paged_attention_prompt_forward(wide[:, 256:256 + heads * 128], kp, vp, ks, vs, table[:, :7], lengths, cu, scale=0.3), a)


def test_a_sequence_does_not_depend_on_its_batch():
    lengths = [1, 900, 5000, 64, 2049, 1024]
    cache = Cache(lengths, 2, 128, 64, seed=12)
    q = queries(6, 16, 128, BF).to(DEV)
    kp, vp, ks, vs, table, held = cache.device()
    together = K.paged_attention_decode_forward(q, kp, vp, ks, vs, table, held)
    assert torch.equal(together, K.paged_attention_decode_forward(q, kp, vp, ks, vs, table, held))
    for s in range(6):
        alone = K.paged_attention_decode_forward(q[s:s + 1], kp, vp, ks, vs, table[s:s + 1], held[s:s + 1])
        narrow = K.paged_attention_decode_forward(q[s:s + 1], kp, vp, ks, vs, table[s:s + 1, :-(-lengths[s] // 64)], held[s:s + 1])
        assert torch.equal(alone[0], together[s]) and torch.equal(narrow[0], together[s])


def test_a_prompt_does_not_depend_on_what_the_others_hold():
    """The same call with other queries and another cache in the other sequences: equal bits."""
    lengths, steps = [1, 900, 5000, 64, 2049, 17], [1, 200, 333, 64, 49, 17]
    cache = Cache(lengths, 2, 128, 64, seed=12)
    cu = torch.tensor([0] + list(np.cumsum(steps)), dtype=torch.int32, device=DEV)
    q = queries(sum(steps), 16, 128, BF).to(DEV)
    kp, vp, ks, vs, table, held = cache.device()
    together = K.paged_attention_prompt_forward(q, kp, vp, ks, vs, table, held, cu)
    assert torch.equal(together, K.paged_attention_prompt_forward(q, kp, vp, ks, vs, table, held, cu))
    for s in range(6):
        other_q, other_k, other_held = torch.randn_like(q), torch.full_like(kp.view(torch.uint8), 0x30), torch.ones_like(held)
        other_q[cu[s]:cu[s + 1]] = q[cu[s]:cu[s + 1]]
        pages = table[s, :-(-lengths[s] // 64)].long()
        other_k[pages] = kp.view(torch.uint8)[pages]
        other_held[s] = held[s]
        got = K.paged_attention_prompt_forward(other_q, other_k, vp.view(torch.uint8), ks, vs, table, other_held, cu)
        assert torch.equal(got[cu[s]:cu[s + 1]], together[cu[s]:cu[s + 1]])


# few rows before a long context: the keys in runs, some of them empty for a short sequence beside a long one
@pytest.mark.parametrize("steps,pasts,heads,kv_heads,dim,page,dtype", [
    ([3], [3100], 6, 1, 128, 64, BF), ([1, 300, 10, 11, 1, 0, 2], [1500, 700, 1024, 3, 0, 0, 5000], 6, 1, 128, 32, BF), ([1] * 70 + [90], list(range(1000, 1070)) + [30], 2, 2, 64, 64, HF),
    ([64, 65, 8], [1100, 1100, 4000], 1, 1, 128, 16, HF), ([33], [1200], 2, 1, 128, 64, BF), ([1, 2, 40], [1500, 2000, 100], 32, 1, 64, 32, BF), ([1, 3], [3000, 100], 128, 1, 64, 64, HF), ([32], [1200], 2, 1, 128, 64, BF), ([40, 2, 0, 1], [2000, 0, 0, 4095], 2, 1, 64, 16, HF), ([17, 70], [5000, 10], 8, 2, 128, 128, HF), ([1], [9000], 16, 2, 64, 32, BF)])
def test_prompt_in_runs_against_float64(steps, pasts, heads, kv_heads, dim, page, dtype):
    cache = Cache([n + p if n else 0 for n, p in zip(steps, pasts)], kv_heads, dim, page, seed=sum(steps) + heads)
    cu = np.concatenate([[0], np.cumsum(steps)])
    q = queries(cu[-1] + 5, heads, dim, dtype, seed=2)
    lib = _ffi.load_library()
    assert lib.pllm_paged_attention_prompt_workspace_bytes(cu[-1] + 5, len(steps), heads, kv_heads, dim, cache.width * page) > 0, "the case has one run"
    if steps[0] == 17:
        cache.table[0, 5] = -1
    got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
    want, note = cache.attention(q[:cu[-1]].view(-1, heads, dim).double().numpy(), cu)
    close(got[:cu[-1]], want, note, dtype)
    assert (got[cu[-1]:] == 0).all()


# Calls of many rows and heads, of which a few heads are checked (and one of few rows, in runs): one prompt whose workgroups are up to twice the compute units, the same behind a past, two long
# runs of the keys, ragged ones, more sequences than a wave has lanes with several blocks in some.
@pytest.mark.parametrize("steps,pasts,kv_heads,group,dim,page,dtype", [
    ([20, 30], [600, 900], 2, 3, 128, 64, BF), ([700], [0], 64, 1, 64, 64, BF), ([600], [700], 64, 1, 128, 32, HF), ([300], [4200], 64, 1, 64, 128, BF), ([290, 1, 310], [100, 900, 700], 64, 1, 128, 32, BF),
    ([3] * 69 + [700, 0, 300], [10] * 69 + [0, 0, 200], 16, 2, 64, 16, HF)])
def test_calls_of_many_rows(steps, pasts, kv_heads, group, dim, page, dtype):
    """NaN values: of the first sequence's sixth key in one dimension, of the last one's last key (one query sees it) in another."""
    lengths = [n + p if n else 0 for n, p in zip(steps, pasts)]
    cache = Cache(lengths, kv_heads, dim, page, seed=sum(steps))
    cache.value_codes[cache.table[0, 0], :, 7, 5] = 0x7f
    cache.value_codes[cache.table[-1, (lengths[-1] - 1) // page], :, 30, (lengths[-1] - 1) % page] = 0xff
    cu = np.concatenate([[0], np.cumsum(steps)])
    q = queries(cu[-1], kv_heads * group, dim, dtype, seed=3)
    got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV)).view(-1, kv_heads, group, dim)
    for head in (0, kv_heads - 1):
        want, note = P.attention(q.view(-1, kv_heads, group, dim)[:, head].double().numpy(), *(a[:, head:head + 1] for a in (
            cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales)), cache.table, cache.lengths, cu, dim ** -0.5)
        assert np.isnan(want).sum() == group * (min(steps[0], lengths[0] - 5) + 1)
        close(got[:, head], want, note, dtype)


def test_many_sequences():
    """More sequences than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(3)
    steps = [int(n) for n in rng.integers(0, 4, 150)]
    lengths = [n + int(p) if n else 0 for n, p in zip(steps, rng.integers(0, 40, 150))]
    cache = Cache(lengths, 1, 64, 16, seed=13)
    cu = np.concatenate([[0], np.cumsum(steps)])
    q = queries(cu[-1], 3, 64, HF)
    got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
    close(got, *cache.attention(q.view(-1, 3, 64).double().numpy(), cu), HF)
    q = queries(150, 3, 64, HF)
    close(_decode(cache, q), *cache.attention(q.view(-1, 3, 64).double().numpy(), _even(150, 1)), HF)


@pytest.mark.parametrize("steps,pasts,heads,kv_heads,dim,page,dtype", [
    ([1, 2, 1, 0, 1], [500, 30, 0, 0, 900], 6, 1, 128, 64, BF), ([1] * 40 + [9, 0, 1], list(range(0, 800, 20)) + [300, 0, 5], 12, 4, 64, 32, HF),
    ([1, 1, 40] * 12, [100, 0, 70] * 12, 16, 16, 64, 16, BF)])
def test_short_sequences_before_narrow_tables(steps, pasts, heads, kv_heads, dim, page, dtype):
    """Few rows in all, mostly short ones of many sequences and heads, rows behind the last."""
    cache = Cache([n + p if n else 0 for n, p in zip(steps, pasts)], kv_heads, dim, page, seed=sum(steps))
    cu = np.concatenate([[0], np.cumsum(steps)])
    q = queries(cu[-1] + 3, heads, dim, dtype, seed=4)
    got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
    close(got[:cu[-1]], *cache.attention(q[:cu[-1]].view(-1, heads, dim).double().numpy(), cu), dtype)
    assert (got[cu[-1]:] == 0).all()


def test_no_sequences_and_no_tokens():
    cache = Cache([10], 1, 64, 16)
    kp, vp, ks, vs, table, lengths = cache.device()
    q = torch.zeros(0, 128, dtype=BF, device=DEV)
    assert K.paged_attention_decode_forward(q, kp, vp, ks, vs, table[:0], lengths[:0]).shape == (0, 128)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert K.paged_attention_prompt_forward(q, kp, vp, ks, vs, table, lengths, torch.zeros(2, dtype=torch.int32, device=DEV)).shape == (0, 128)
    assert (K.paged_attention_prompt_forward(torch.ones(3, 128, dtype=BF, device=DEV), kp, vp, ks, vs, table[:0], lengths[:0], none) == 0).all()


def test_offsets_of_any_kind_stay_inside_the_rows():
    """Offsets that are no offsets (falling, negative, beyond the rows): which rows are computed is not defined, that the call ends and the rows of
    sequences in order are right is."""
    cache = Cache([20, 20, 20], 1, 64, 16, seed=14)
    q = queries(60, 2, 64, BF).to(DEV)
    for cu in ([0, 20, -7, 60], [0, 1000, 1000, 1000], [0, 20, 10, 5], [5, 20, 40, 60]):
        got = K.paged_attention_prompt_forward(q, *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        assert got.shape == q.shape


def test_pages_behind_four_gigabytes():
    """Codes at byte offsets past 32 bits."""
    dim, page, kv_heads = 128, 128, 8
    pool = (1 << 32) // (dim * page * kv_heads) + 8
    cache = Cache([300], kv_heads, dim, page, seed=15, spare=1)
    kp = torch.empty(pool, kv_heads, page, dim, dtype=torch.uint8, device=DEV)
    vp = torch.empty(pool, kv_heads, dim, page, dtype=torch.uint8, device=DEV)
    ks, vs = torch.empty(pool, kv_heads, device=DEV), torch.empty(pool, kv_heads, device=DEV)
    small = cache.device()
    shift = pool - cache.pool
    for big, part in ((kp, small[0].view(torch.uint8)), (vp, small[1].view(torch.uint8)), (ks, small[2]), (vs, small[3])):
        big[shift:] = part
    table = small[4] + shift
    q = queries(1, 16, dim, BF).to(DEV)
    assert torch.equal(K.paged_attention_decode_forward(q, kp, vp, ks, vs, table, small[5]), K.paged_attention_decode_forward(q, *small))
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    assert torch.equal(K.paged_attention_prompt_forward(q, kp, vp, ks, vs, table, small[5], cu), K.paged_attention_prompt_forward(q, *small, cu))


def test_captured_twice_and_replayed_on_other_lengths():
    """Two captured graphs (each with a workspace of its own), replayed in turn and beside eager calls, lengths and pages changed in between."""
    lengths = [900, 3000, 64, 1]
    cache = Cache(lengths, 2, 128, 64, seed=16)
    kp, vp, ks, vs, table, held = cache.device()
    q = queries(4, 12, 128, BF).to(DEV)
    cu = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=DEV)
    args = (kp, vp, ks, vs, table, held)
    K.paged_attention_decode_forward(q, *args)
    graphs, outs = [], []
    for form in (lambda: K.paged_attention_decode_forward(q, *args), lambda: K.paged_attention_decode_forward(q, *args), lambda: K.paged_attention_prompt_forward(q, *args, cu)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(form())
        graphs.append(graph)
    for seed, now in ((1, lengths), (2, [1, 17, 64, 0]), (3, [700, 2999, 63, 1]), (4, lengths)):
        q.copy_(queries(4, 12, 128, BF, seed=seed).to(DEV))
        held.copy_(torch.tensor(now, dtype=torch.int32, device=DEV))
        for g in graphs:
            g.replay()
        eager = K.paged_attention_decode_forward(q, *args)
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
        assert torch.equal(outs[2], K.paged_attention_prompt_forward(q, *args, cu))
        torch.cuda.synchronize()


def test_two_streams_at_once():
    cache = Cache([2500, 800], 4, 128, 64, seed=17)
    args = cache.device()
    qs = [queries(2, 16, 128, BF, seed=i).to(DEV) for i in range(2)]
    want = [K.paged_attention_decode_forward(q, *args) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(K.paged_attention_decode_forward(qs[i], *args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_prompts_in_runs_captured_and_on_two_streams_at_once():
    """Workspaces between two launches: captured graphs replayed in turn on other lengths and offsets, and eager calls on two streams, against calls alone."""
    cache = Cache([2500, 800, 1900], 2, 128, 64, seed=18)
    args = cache.device()
    held = args[5]
    qs = [queries(120, 12, 128, BF, seed=i).to(DEV) for i in range(2)]
    cu = torch.tensor([0, 70, 71, 110], dtype=torch.int32, device=DEV)
    assert _ffi.load_library().pllm_paged_attention_prompt_workspace_bytes(120, 3, 12, 2, 128, cache.width * 64) > 0
    want = [K.paged_attention_prompt_forward(q, *args, cu) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(K.paged_attention_prompt_forward(qs[i], *args, cu))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            outs.append(K.paged_attention_prompt_forward(qs[i], *args, cu))
    for lengths, offsets in (([2500, 800, 1900], [0, 70, 71, 110]), ([70, 1, 40], [0, 70, 71, 110]), ([1000, 0, 1800], [0, 5, 5, 120]), ([2400, 790, 1000], [0, 1, 100, 101])):
        held.copy_(torch.tensor(lengths, dtype=torch.int32, device=DEV))
        cu.copy_(torch.tensor(offsets, dtype=torch.int32, device=DEV))
        for graph in graphs:
            graph.replay()
        for i in range(2):
            assert torch.equal(outs[i], K.paged_attention_prompt_forward(qs[i], *args, cu)) and bool((outs[i][offsets[-1]:] == 0).all())
        torch.cuda.synchronize()
