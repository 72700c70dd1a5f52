"""Attention over the paged E4M3 cache in fp16 where a few keys hold almost all of a row's weight: what the many others add up to is not lost with the 16 bits that a
weight is rounded to, and a weight never passes fp16's largest value."""
import numpy as np
import pytest
import torch

from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
DEV, HF = "cuda:0", torch.float16
F8 = torch.float8_e4m3fn


def _paged(keys, values, page, value_scale=1.0):
    """keys, values [kv_heads, positions, dim] (E4M3 values) of one sequence as a cache, its pages in order."""
    kv_heads, positions, dim = keys.shape
    pages = -(-positions // page)
    blank = torch.zeros(kv_heads, pages * page - positions, dim, device=DEV)
    keys, values = (torch.cat([t, blank], 1).view(kv_heads, pages, page, dim).transpose(0, 1) for t in (keys, values))
    return (keys.contiguous().to(F8), values.transpose(2, 3).contiguous().to(F8), torch.ones(pages, kv_heads, device=DEV), torch.full((pages, kv_heads), value_scale, device=DEV),
            torch.arange(pages, dtype=torch.int32, device=DEV)[None].contiguous(), torch.tensor([positions], dtype=torch.int32, device=DEV))


def _check(got, first, keys, values, visible, room):
    """got [heads of one key/value head, dim]; scores are first[head] * keys[:, 0].

    Weights and the output are rounded as elsewhere (u = 2^-11 of the weighted mean of |v| once above and once below the division, of the output once; float32 sums of `keys` terms
    in four or more chains and 80 other roundings).  A weight that is no normal fp16 number is off by up to 2^-25 where the row's largest is 2^room at least: 2^-(25 + room) of it,
    above and below the division."""
    k, v = keys[:visible, 0].double().cpu(), values[:visible].double().cpu()
    score = first.double().cpu()[:, None] * k[None]
    w = torch.exp(score - score.amax(1, keepdim=True))
    den = w.sum(1, keepdim=True)
    want, spread, top = w @ v / den, w @ v.abs() / den, v.abs().amax() / den
    u, f32 = 2.0 ** -11, (score.abs().amax(1, keepdim=True) * 12 + 80 + visible / 16) * 2.0 ** -24
    bound = u * (spread + 2 * want.abs()) * (1 + 3 * u) + 2 * f32 * (spread + want.abs()) + 2.0 ** -(24 + room) * visible * top + 2.0 ** -25
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.1f} bounds, {float((off / want.abs()).max()):.4f} of the value"


def _tail(kv_heads, positions, dim, sinks, seed):
    """Keys with one value in their first dimension: 2.25 in those that hold the weight, 0.171875 - 0.203125 in the rest; values of mean one, of the former zero."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    keys = torch.zeros(kv_heads, positions, dim, device=DEV)
    keys[:, :, 0] = 0.171875 + 0.015625 * torch.randint(0, 3, (kv_heads, positions), generator=g, device=DEV).float()
    keys[:, sinks, 0] = 2.25
    values = 1.0 + 0.125 * torch.randint(-7, 8, (kv_heads, positions, dim), generator=g, device=DEV).float()
    values[:, sinks] = 0.0
    return keys, values.to(F8).float()


def _first(heads, dim, rows):
    """Queries with one value in their first dimension: 8 up to 10 by head, so 16 to 21 nats between the two kinds of keys."""
    q = torch.zeros(rows, heads, dim, device=DEV)
    q[:, :, 0] = 8.0 + torch.arange(heads, device=DEV) % 64 / 32
    return q


# (tokens, positions, heads, dim, page, the keys that hold the weight): blocks of 256 rows; of 128, whose waves have half of each tile's keys
@pytest.mark.parametrize("tokens,positions,heads,dim,page,sinks", [(520, 33001, 64, 64, 64, [0]), (520, 33001, 64, 128, 128, [70, 71]), (8192, 8192, 4, 64, 16, [0, 32])])
def test_prompt_keeps_what_many_small_weights_add_up_to(tokens, positions, heads, dim, page, sinks):
    keys, values = _tail(1, positions, dim, sinks, 1)
    q = _first(heads, dim, tokens)
    got = K.paged_attention_prompt_forward(q.view(tokens, -1).to(HF), *_paged(keys, values, page), torch.tensor([0, tokens], dtype=torch.int32, device=DEV), scale=1.0)
    for t in (tokens - 1, tokens - 130, tokens // 2):
        _check(got.view(tokens, heads, dim)[t], q[t, :, 0], keys[0], values[0], positions - tokens + t + 1, 11)


@pytest.mark.parametrize("heads,steps,dim,page", [(64, 1, 64, 64), (256, 5, 64, 128)])
def test_decode_keeps_what_many_small_weights_add_up_to(heads, steps, dim, page):
    """Runs of 4096 keys, of which a wave has 64 of every 256."""
    positions, kv_heads = 32768, 64
    keys, values = _tail(kv_heads, positions, dim, [4096 * r + 64 * w for r in range(8) for w in range(4)], 2)
    q = _first(heads, dim, steps)
    got = K.paged_attention_decode_forward(q.view(1, steps, -1).to(HF), *_paged(keys, values, page, 64.0), scale=1.0).view(steps, kv_heads, heads // kv_heads, dim)
    for head in (0, 31, 63):
        for t in {0, steps - 1}:
            _check(got[t, head].float() / 64, q.view(steps, kv_heads, -1, dim)[t, head, :, 0], keys[head], values[head], positions - steps + t + 1, 15)


# (tokens, heads): the decode form; prompts in blocks of 128 and of 256 rows, the latter's earlier tokens without a position
@pytest.mark.parametrize("tokens,heads", [(1, 2), (70, 2), (560, 128)])
def test_scores_that_float32_holds_in_steps_of_sixteen(tokens, heads):
    """Scores of 2^27 + 16 and 2^27 + 32 (to base 2): the larger key has all the weight but 2^-16; a weight of 2^16 would be fp16's infinity."""
    scale = np.float32(0.6931472)
    assert np.float32(scale * np.float32(1.4426950408889634)) == 1.0
    keys, values = torch.zeros(1, 200, 64, device=DEV), torch.ones(1, 200, 64, device=DEV)
    keys[:, :, 0], keys[:, 20, 1], keys[:, 100, 1] = 256.0, 1.0, 2.0
    values[:, 100] = 3.0
    kp, vp, ks, vs, table, lengths = _paged(keys, values, 16)
    ks.fill_(16.0)
    q = torch.zeros(tokens, heads, 64, device=DEV)
    q[:, :, 0], q[:, :, 1] = 32768.0, 1.0
    q = q.view(tokens, -1).to(HF)
    if tokens == 1:
        got = K.paged_attention_decode_forward(q, kp, vp, ks, vs, table, lengths, scale=float(scale))
    else:
        cu = torch.tensor([0, tokens], dtype=torch.int32, device=DEV)
        got = K.paged_attention_prompt_forward(q, kp, vp, ks, vs, table, lengths, cu, scale=float(scale))
    assert bool(((got[-60:] - 3.0).abs() <= 3 * 2.0 ** -10).all()), got[-1, :4]
