"""Appending to the paged E4M3 cache against a float64 form.

Values: no arithmetic before the quantization and power-of-two scales, so codes and scales are equal.  Queries turned in float32: x cos + y sin
with one rounding of the product and one of the fused sum, so off by at most 2^-23 (|x cos| + |y sin|); keys in 64 bits, held to the same; a key's code lies between those of the two
ends, a page's scale between theirs, and a query is within half a step of its type of a value between them."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import DEV, Cache
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _rows(tokens, width, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, width, generator=g) * torch.exp(spread * torch.randn(tokens, 1, generator=g))).to(dtype)


def _between(got, lo, hi):
    return np.all(((got >= lo) & (got <= hi)) | (np.isnan(got) & np.isnan(lo)))


def _check(cache, before, after, q_out, q, k, v, cu, rope, cos, sin, heads):
    """`before`: the host arrays as they were; `after`: the device tensors."""
    dim, kv_heads = cache.dim, cache.kv_heads
    codes = [after[0].view(torch.uint8).cpu().numpy(), after[1].view(torch.uint8).cpu().numpy()]
    scales = [after[2].cpu().numpy().astype(np.float64), after[3].cpu().numpy().astype(np.float64)]
    tokens = k.shape[0]
    first = np.array([n - (cu[s + 1] - cu[s]) for s, n in enumerate(cache.lengths)])
    seq = np.array([max(s for s in range(len(cu) - 1) if cu[s] <= i) for i in range(cu[-1])], dtype=int)
    pos = np.array([first[s] + i - cu[s] for i, s in enumerate(seq)], dtype=int)
    placed = (pos >= 0) & (pos < cache.width * cache.page)
    at = np.clip(pos, 0, cache.width * cache.page - 1)

    def turned(x):
        x = x[:cu[-1]].float().numpy().astype(np.float64).reshape(cu[-1], -1, dim)
        if not rope:
            return x, np.zeros_like(x)
        return P.turn(x, cos[at], sin[at], rope), 2.0 ** -23 * P.turn(np.abs(x), np.abs(cos[at]), np.abs(sin[at]), rope)

    keys, off = turned(k)
    values = v.float().numpy().astype(np.float64).reshape(tokens, kv_heads, dim)
    lo = P.append(keys - np.sign(keys) * off, values, *before, cache.table, cache.lengths, cu)
    hi = P.append(keys + np.sign(keys) * off, values, *before, cache.table, cache.lengths, cu)
    used = np.zeros(cache.pool, dtype=bool)
    for s, p in zip(seq[placed], pos[placed] // cache.page):
        if 0 <= cache.table[s, p] < cache.pool:
            used[cache.table[s, p]] = True
    # values: equal codes (as what they stand for; the sign of a zero too) and scales
    got = P.e4m3_decode(codes[1])
    assert np.array_equal(got, lo[1], equal_nan=True) and np.array_equal(scales[1], lo[3], equal_nan=True)
    # keys: between the ends; magnitudes grow with the scale's choice, so compare where both ends chose the same
    got = P.e4m3_decode(codes[0])
    assert _between(scales[0][used], lo[2][used], hi[2][used])
    same = lo[2][used] == hi[2][used]
    a, b = np.minimum(lo[0], hi[0])[used], np.maximum(lo[0], hi[0])[used]
    assert _between(got[used][same], a[same], b[same])
    # pages that no token went to are as they were
    assert np.array_equal(codes[0][~used], before[0][~used]) and np.array_equal(codes[1][~used], before[1][~used])
    assert np.array_equal(scales[0][~used], before[2][~used], equal_nan=True) and np.array_equal(scales[1][~used], before[3][~used], equal_nan=True)
    if q is not None:
        want, off = turned(q)
        got = q_out.cpu().double().numpy().reshape(tokens, heads, dim)
        u = torch.finfo(q.dtype).eps / 2
        assert (np.abs(got[:cu[-1]] - want)[placed] <= (off + u * (np.abs(want) + off) + 2.0 ** -25)[placed]).all()
        if rope:
            assert (got[:cu[-1]][~placed] == 0).all() and (got[cu[-1]:] == 0).all()


def _run(steps, pasts, heads, kv_heads, dim, page, rope, dtype, seed=0, even=False, extra=0, change=None, spread=1.0, width=None):
    cache = Cache([n + p for n, p in zip(steps, pasts)], kv_heads, dim, page, seed=seed, width=width)
    if change:
        change(cache)
    cu = np.concatenate([[0], np.cumsum(steps)])
    tokens = cu[-1] + extra
    q, k, v = (_rows(tokens, w * dim, dtype, seed + i, spread) for i, w in enumerate((heads, kv_heads, kv_heads)))
    cos, sin = P.rotary_rows(cache.width * page, dim, rope) if rope else (None, None)
    before = [a.copy() for a in (cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales)]
    args = cache.device()
    out = K.paged_kv_append_forward(q.to(DEV), k.to(DEV), v.to(DEV), *args, cu_steps=None if even else torch.tensor(cu, dtype=torch.int32, device=DEV),
                                    cos_table=torch.from_numpy(cos).to(DEV) if rope else None, sin_table=torch.from_numpy(sin).to(DEV) if rope else None, rope_dim=rope)
    torch.cuda.synchronize()
    _check(cache, before, args, out, q, k, v, cu, rope, cos, sin, heads)
    return cache, args, out


# (steps, pasts, heads, kv_heads, dim, page, rope, dtype)
CASES = [
    ([1], [0], 1, 1, 64, 16, 64, BF), ([1, 1, 1, 1], [0, 15, 16, 63], 6, 1, 128, 16, 64, HF), ([5, 17, 1], [14, 0, 31], 4, 2, 128, 32, 128, BF),
    ([64, 65, 63], [0, 0, 1], 48, 8, 128, 64, 64, BF), ([130, 3, 200], [0, 125, 77], 5, 5, 64, 128, 32, HF), ([33], [100], 16, 2, 128, 128, 96, BF),
    ([100, 50], [7, 60], 2, 2, 128, 16, 16, HF), ([40], [0], 8, 1, 64, 64, 0, BF), ([7, 0, 9], [3, 0, 20], 3, 1, 64, 32, 48, BF),
    ([i % 4 for i in range(130)], [(7 * i) % 40 if i % 4 else 0 for i in range(130)], 3, 1, 128, 16, 64, BF), ([0, 0, 5] * 30, [0, 0, 9] * 30, 17, 1, 128, 32, 128, HF),
]


@pytest.mark.parametrize("steps,pasts,heads,kv_heads,dim,page,rope,dtype", CASES)
def test_against_float64(steps, pasts, heads, kv_heads, dim, page, rope, dtype):
    _run(steps, pasts, heads, kv_heads, dim, page, rope, dtype, seed=sum(steps))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_keys_codes_are_those_of_the_exact_values(dtype):
    """Turned keys are two exact products and one sum in 64 bits: off by 2^-52 of the products at most."""
    steps, dim, page, kv_heads, rope = [700, 500], 128, 64, 4, 128
    cache, args, _ = _run(steps, [0, 0], 4, kv_heads, dim, page, rope, dtype, seed=8)
    cos, sin = P.rotary_rows(cache.width * page, dim, rope)
    pos = np.concatenate([np.arange(n) for n in steps])
    k = _rows(sum(steps), kv_heads * dim, dtype, 9).float().numpy().astype(np.float64).reshape(-1, kv_heads, dim)
    turned, off = P.turn(k, cos[pos], sin[pos], rope), 2.0 ** -52 * P.turn(np.abs(k), np.abs(cos[pos]), np.abs(sin[pos]), rope)
    got, scales, at = P.e4m3_decode(args[0].view(torch.uint8).cpu().numpy()), args[2].cpu().numpy().astype(np.float64), 0
    for s, n in enumerate(steps):
        for p in range(-(-n // page)):
            which, rows = cache.table[s, p], slice(at + p * page, at + min(n, (p + 1) * page))
            v, e = turned[rows].transpose(1, 0, 2), off[rows].transpose(1, 0, 2)
            scale = P.page_scale(np.abs(v).max((1, 2)))
            assert np.array_equal(scales[which], scale)
            lo, hi = P.e4m3_round((v - e) / scale[:, None, None]), P.e4m3_round((v + e) / scale[:, None, None])
            mine = got[which][:, :v.shape[1]]
            assert ((mine >= lo) & (mine <= hi)).all()
        at += n


def test_even_steps_without_offsets():
    _run([3] * 70, [int(p) for p in np.random.default_rng(0).integers(0, 90, 70)], 4, 2, 128, 32, 64, BF, seed=3, even=True)


@pytest.mark.parametrize("steps,heads,kv_heads,dim,page", [(1, 48, 8, 128, 64), (4, 5, 1, 128, 16), (5, 17, 1, 128, 128), (8, 33, 1, 64, 32), (9, 2, 2, 64, 16), (1, 130, 2, 64, 128)])
def test_even_steps_of_one_wave_and_more(steps, heads, kv_heads, dim, page):
    """Four tokens of 128-wide heads, eight of 64-wide ones are one wave's; heads beyond one workgroup's share."""
    pasts = [0, 1, page - 1, page, 3 * page - 2, 2 * page - steps if steps < 2 * page else 0]
    _run([steps] * 6, pasts, heads, kv_heads, dim, page, 32, BF if steps % 2 else HF, seed=steps, even=True, spread=2.0)


def test_rows_behind_the_last_sequence_store_nothing():
    _, _, out = _run([4, 6], [0, 29], 2, 1, 128, 16, 32, BF, extra=9)
    assert (out[10:] == 0).all()


def test_scales_that_rise_take_the_older_codes_along():
    """Tokens one by one, each larger than the page's first: the page is scaled down again and again, to the bits that one append after the
    other gives in the float64 form."""
    dim, page, kv_heads = 64, 32, 2
    cache = Cache([1], kv_heads, dim, page, seed=4, width=2)
    before = [a.copy() for a in (cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales)]
    args = cache.device()
    g = torch.Generator().manual_seed(5)
    host = before
    for i in range(40):
        x = (torch.randn(1, kv_heads * dim, generator=g) * 2.0 ** (i / 3 - 8)).to(BF)
        y = (torch.randn(1, kv_heads * dim, generator=g) * 2.0 ** (8 - i / 3)).to(BF)
        args[5].fill_(i + 1)
        K.paged_kv_append_forward(None, x.to(DEV), y.to(DEV), *args)
        rows = [t.double().numpy().reshape(1, kv_heads, dim) for t in (x, y)]
        out = P.append(*rows, *host, cache.table, [i + 1], [0, 1])
        got = [args[0].view(torch.uint8).cpu().numpy(), args[1].view(torch.uint8).cpu().numpy(), args[2].cpu().numpy(), args[3].cpu().numpy()]
        assert np.array_equal(P.e4m3_decode(got[0]), out[0], equal_nan=True) and np.array_equal(P.e4m3_decode(got[1]), out[1], equal_nan=True), i
        assert np.array_equal(got[2], out[2], equal_nan=True) and np.array_equal(got[3], out[3], equal_nan=True), i
        host = got


def test_the_same_call_again_changes_nothing():
    steps, pasts = [20, 1, 70], [5, 64, 0]
    cache = Cache([n + p for n, p in zip(steps, pasts)], 2, 128, 32, seed=6)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(steps)]), dtype=torch.int32, device=DEV)
    k, v = (_rows(91, 256, HF, s).to(DEV) for s in (1, 2))
    args = cache.device()
    K.paged_kv_append_forward(None, k, v, *args, cu_steps=cu)
    once = [t.clone() for t in args]
    K.paged_kv_append_forward(None, k, v, *args, cu_steps=cu)
    for a, b in zip(args, once):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_zeros_largest_values_and_what_is_not_finite():
    cache = Cache([16, 16, 16], 1, 64, 16, seed=7)
    k = torch.zeros(48, 64, dtype=BF)
    v = torch.zeros(48, 64, dtype=BF)
    k[16:32], v[16:32] = torch.finfo(BF).max, -torch.finfo(BF).max
    k[32, 0], k[33, 1], v[40, 2], v[41, 3], k[34, 5], v[42, 6] = float("inf"), float("nan"), float("-inf"), float("nan"), 7.0, -3.5
    args = cache.device()
    K.paged_kv_append_forward(None, k.to(DEV), v.to(DEV), *args)
    ids = cache.table[:, 0]
    kc, vc, ks, vs = args[0].float().cpu()[ids], args[1].float().cpu()[ids].transpose(2, 3), args[2].cpu()[ids], args[3].cpu()[ids]
    assert (kc[0] == 0).all() and (vc[0] == 0).all() and float(ks[0]) == 2.0 ** -120 == float(vs[0])
    assert (kc[1] * 2.0 ** -20 * float(ks[1]) == torch.finfo(BF).max * 2.0 ** -20 / (255 / 256)).all()      # 2^128 over 2^20: the nearest code's value
    assert (vc[1] == -kc[1]).all() and float(vs[1]) == float(ks[1])
    assert kc[2, 0, 0, 0].isnan() and kc[2, 0, 1, 1].isnan() and float(ks[2]) == 2.0 ** -6 and float(kc[2, 0, 2, 5]) == 448.0
    assert vc[2, 0, 8, 2].isnan() and vc[2, 0, 9, 3].isnan() and float(vs[2]) == 2.0 ** -7 and float(vc[2, 0, 10, 6]) == -448.0
    assert int(kc.isnan().sum()) == 2 and int(vc.isnan().sum()) == 2


def test_pages_that_are_missing_and_positions_beyond_the_table():
    def change(cache):
        cache.table[0, 1], cache.table[1, 0] = -3, cache.pool
        cache.lengths[2] = cache.width * cache.page + 5                       # the last five tokens have no place
    _run([40, 8, 30], [0, 0, 10], 4, 2, 64, 16, 32, BF, seed=8, change=change)

    def shorter(cache):
        cache.lengths[:] = [3, -2, 0]                                         # fewer positions than new tokens: the last tokens' positions count
    _run([10, 4, 2], [0, 0, 0], 2, 1, 128, 16, 64, HF, seed=9, change=shorter)


def test_rows_of_a_fused_projection_and_far_positions():
    dim, kv_heads, heads, page = 128, 2, 6, 64
    past = 70000
    cache = Cache([1], kv_heads, dim, page, seed=10, width=-(-(past + 3) // page), spare=4)
    cache.table[0, past // page] = 1
    cache.lengths[0] = past + 3
    cos, sin = (torch.from_numpy(t).to(DEV) for t in P.rotary_rows(cache.width * page, dim, dim))
    wide = _rows(3, (heads + 2 * kv_heads) * dim, BF, 11)
    a, b = heads * dim, (heads + kv_heads) * dim
    fused = wide.to(DEV)
    one, two = cache.device(), cache.device()
    q1 = K.paged_kv_append_forward(fused[:, :a], fused[:, a:b], fused[:, b:], *one, cos_table=cos, sin_table=sin, rope_dim=dim)
    q2 = K.paged_kv_append_forward(fused[:, :a].contiguous(), fused[:, a:b].contiguous(), fused[:, b:].contiguous(), *two, cos_table=cos, sin_table=sin, rope_dim=dim)
    assert torch.equal(q1, q2)
    for x, y in zip(one, two):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    x = wide[:, :a].double().numpy().reshape(3, heads, dim)
    at = np.arange(past, past + 3)
    want = P.turn(x, cos.cpu().numpy()[at], sin.cpu().numpy()[at], dim)
    assert (np.abs(q1.cpu().double().numpy().reshape(want.shape) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -22 * np.abs(x).max() * 2).all()


def test_captured_and_replayed():
    """A decode step's append in a graph: lengths, tables and rows change between replays, eager calls on another copy of the cache say what should come."""
    cache = Cache([10, 31, 64], 2, 128, 32, seed=12, width=8, spare=24)
    free = [p for p in range(1, cache.pool) if p not in set(cache.table.ravel())]
    for s in range(3):
        for p in range(8):
            if cache.table[s, p] >= cache.pool:
                cache.table[s, p] = free.pop() if free else -1
    cos, sin = (torch.from_numpy(t).to(DEV) for t in P.rotary_rows(8 * 32, 128, 64))
    held, eager = cache.device(), cache.device()
    q, k, v = (_rows(3, w * 128, BF, 1).to(DEV) for w in (4, 2, 2))
    call = lambda args: K.paged_kv_append_forward(q, k, v, *args, cos_table=cos, sin_table=sin, rope_dim=64)
    side = cache.device()
    call(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held)
    for i in range(5):
        for t, w in ((q, 4), (k, 2), (v, 2)):
            t.copy_(_rows(3, w * 128, BF, 20 + i + w).to(DEV))
        for t in (held[5], eager[5]):
            t.copy_(torch.tensor([10 + i, 31 + i, 64 + i], dtype=torch.int32, device=DEV) + 1)
        graph.replay()
        want = call(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(held[:4], eager[:4]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
