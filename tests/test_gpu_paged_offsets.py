"""Offsets of the new tokens' rows that are none (falling, negative, beyond the rows) at the C entries: rows that one sequence alone has are right, nothing outside of outputs and
of the tables' pages is written."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import DEV, Cache, close, queries
from pocketllm_amd import _ffi, hip_kernel as K

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ROWS, HEADS, DIM, PAGE = 60, 2, 64, 16
OFFSETS = [[0, 20, -7, 60], [0, 1000, 1000, 1000], [0, 20, 10, 5], [5, 20, 40, 60], [0, 20, 2**31 - 1, 2**31 - 1], [-3, 20, 40, 50]]


def _cut(cu):
    """The rows that each sequence claims (offsets cut to the rows, the first taken as 0) and those that one alone has."""
    at = [0] + [min(max(c, 0), ROWS) for c in cu[1:]]
    claims = [range(a, b) for a, b in zip(at, at[1:])]
    owners = np.zeros(ROWS, dtype=int)
    for c in claims + [range(at[-1], ROWS)]:
        owners[list(c)] += 1
    return at, claims, owners == 1


@pytest.mark.parametrize("cu", OFFSETS)
@pytest.mark.parametrize("width", [2, 300])
def test_prompt(cu, width):
    """A narrow table, and one of 4800 positions: runs of the keys and short sequences by the decode form's kernel."""
    cache = Cache([20, 20, 20], 1, DIM, PAGE, seed=14, width=width)
    q = queries(ROWS, HEADS, DIM, BF).to(DEV)
    guard = 4096
    out = torch.full((guard + ROWS * HEADS * DIM + guard,), 7.0, dtype=BF, device=DEV)
    kp, vp, ks, vs, table, lengths = cache.device()
    offsets = torch.tensor(cu, dtype=torch.int32, device=DEV)
    lib = _ffi.load_library()
    need = lib.pllm_paged_attention_prompt_workspace_bytes(ROWS, 3, HEADS, 1, DIM, width * PAGE)
    assert (need > 0) == (width == 300)
    ws = torch.full((need + 2 * guard,), 0x55, dtype=torch.uint8, device=DEV)
    status = lib.pllm_paged_attention_prompt(q.data_ptr(), HEADS * DIM, 2, kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), cache.pool, PAGE, table.data_ptr(), width, width,
                                             lengths.data_ptr(), offsets.data_ptr(), ROWS, 3, HEADS, 1, DIM, DIM ** -0.5, out[guard:].data_ptr(), ws[guard:].data_ptr() if need else None,
                                             need, torch.cuda.current_stream().cuda_stream)
    assert status == 0
    torch.cuda.synchronize()
    assert bool((out[:guard] == 7).all()) and bool((out[-guard:] == 7).all()) and bool((ws[:guard] == 0x55).all()) and bool((ws[need + guard:] == 0x55).all())
    got = out[guard:-guard].view(ROWS, HEADS * DIM)
    at, claims, alone = _cut(cu)
    assert alone.any()
    for s, claim in enumerate(claims):
        rows = [r for r in claim if alone[r]]
        if rows:
            want, note = P.attention(q[claim.start:claim.stop].view(-1, HEADS, DIM).cpu().double().numpy(), cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales,
                                     cache.table[s:s + 1], cache.lengths[s:s + 1], [0, len(claim)], DIM ** -0.5)
            which = np.array(rows) - claim.start
            close(got[rows], want[which], {n: v[which] for n, v in note.items()}, BF)
    behind = [r for r in range(at[-1], ROWS) if alone[r]]
    assert bool((got[behind] == 0).all())


@pytest.mark.parametrize("cu", OFFSETS)
@pytest.mark.parametrize("heads", [2, 40])
def test_append(cu, heads):
    """Pages that no table names, and slots behind every sequence's end, stay as they are."""
    cache = Cache([20, 20, 20], 2, DIM, PAGE, seed=15, spare=6)
    before = [cache.key_codes.copy(), cache.value_codes.copy(), cache.key_scales.copy(), cache.value_scales.copy()]
    q, k, v = (queries(ROWS, n, DIM, BF, seed=i) for i, n in enumerate((heads, 2, 2)))
    pools = cache.device()
    cos, sin = P.rotary_rows(cache.width * PAGE, DIM, 32)
    guard = 4096
    out = torch.full((guard + ROWS * heads * DIM + guard,), 7.0, dtype=BF, device=DEV)
    dev = [t.to(DEV) for t in (q, k, v, torch.from_numpy(cos), torch.from_numpy(sin), torch.tensor(cu, dtype=torch.int32))]
    status = _ffi.load_library().pllm_paged_kv_append(
        dev[0].data_ptr(), heads * DIM, dev[1].data_ptr(), 2 * DIM, dev[2].data_ptr(), 2 * DIM, 2, out[guard:].data_ptr(), *(t.data_ptr() for t in pools[:4]), cache.pool, PAGE,
        pools[4].data_ptr(), cache.width, cache.width, pools[5].data_ptr(), dev[5].data_ptr(), dev[3].data_ptr(), dev[4].data_ptr(), cache.width * PAGE, 32, ROWS, 3, heads, 2, DIM,
        torch.cuda.current_stream().cuda_stream)
    assert status == 0
    torch.cuda.synchronize()
    assert bool((out[:guard] == 7).all()) and bool((out[-guard:] == 7).all())
    named = np.zeros(cache.pool, dtype=bool)
    named[cache.table[(cache.table >= 0) & (cache.table < cache.pool)]] = True
    assert (~named).sum() == 6
    after = [t.cpu().view(torch.uint8).numpy() if i < 2 else t.cpu().numpy() for i, t in enumerate(pools[:4])]
    for a, b in zip(after, before):
        assert np.array_equal(a[~named], b[~named], equal_nan=a.dtype.kind == "f")
    for s in range(3):                                                        # 20 positions: the second page's slots from its fourth on
        last = cache.table[s, 1]
        assert np.array_equal(after[0][last][:, 4:], before[0][last][:, 4:]) and np.array_equal(after[1][last][:, :, 4:], before[1][last][:, :, 4:])


def test_calls_whose_keys_are_cut_in_runs():
    """The workspace is more than the short sequences' part of it can be: the rest are runs of the others' keys."""
    lib = _ffi.load_library()
    for steps, pasts, heads, kv_heads, dim, page in (([66, 200], [3000, 4000], 2, 1, 64, 64), ([100, 1, 70], [2000, 3000, 100], 4, 2, 128, 32)):
        cache = Cache([n + p for n, p in zip(steps, pasts)], kv_heads, dim, page, seed=sum(steps))
        cu = np.concatenate([[0], np.cumsum(steps)])
        need = lib.pllm_paged_attention_prompt_workspace_bytes(int(cu[-1]), len(steps), heads, kv_heads, dim, cache.width * page)
        assert need > lib.pllm_paged_attention_decode_workspace_bytes(len(steps), 64, kv_heads, kv_heads, dim, cache.width * page)
        q = queries(cu[-1], heads, dim, BF, seed=5)
        got = K.paged_attention_prompt_forward(q.to(DEV), *cache.device(), torch.tensor(cu, dtype=torch.int32, device=DEV))
        close(got, *cache.attention(q.view(-1, heads, dim).double().numpy(), cu), BF)
