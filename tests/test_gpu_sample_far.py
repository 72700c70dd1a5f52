"""sample_tokens_forward where distances from the largest logit leave float32's range, as logits or as numbers of bins: a few allowed tokens beside masked ones, finite logits
farther apart than the largest float32, NaN of any kind."""
import numpy as np
import pytest
import torch

from oracle import tree_oracle as T
from test_gpu_sample import check, sampled

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def both_sides(row, **given):
    """Numbers on both sides of every border between the tokens that are kept of a row, and in the middle between borders."""
    x, params = row.double().numpy(), {n: float(np.float32(v)) for n, v in given.items()}
    params = {n: int(v) if n == "top_k" else v for n, v in params.items()}
    tokens, borders = [], []
    for u in (np.arange(256) + 0.5) / 256:                                    # (no allowed token below has less than 1/256)
        token, _ = T.sample(x, u, **params)
        if not tokens or token != tokens[-1]:
            low, high = (u - 1 / 256, u) if tokens else (0.0, 0.0)
            for _ in range(20 if tokens else 0):
                middle = (low + high) / 2
                low, high = (middle, high) if T.sample(x, middle, **params)[0] != token else (low, middle)
            tokens.append(token)
            borders.append(high)
    borders.append(1.0)
    return sorted({float(np.float32(u)) for a, b in zip(borders, borders[1:]) for u in (a + 1e-5, (a + b) / 2, b - 1e-5)})


PARAMETERS = [dict(), dict(top_p=0.99), dict(top_p=0.6), dict(top_k=1500), dict(top_k=1500, top_p=0.9), dict(min_p=0.05), dict(temperature=0.7, min_p=0.01), dict(top_k=40),
              dict(temperature=3.0, top_p=0.97)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3200, 40000])
@pytest.mark.parametrize("allowed", [{40: 10.0, 41: 8.0}, {40: 2.0, 41: 0.0, 42: -1.0}, {41: -3.0, 42: 1.0, 43: 0.5}, {40: 5.0, 41: 3.0, 800: 5.0, 802: 2.5},
                                     {8: 0.0, 9: -1.75, 1600: 0.0, 1601: -2.0, 3192: 0.0, 3194: -2.5}])
def test_a_few_allowed_tokens(allowed, vocab, dtype):
    """All else is masked: every chunk of 16 bytes that has an allowed token has a masked one too, and the largest of each such chunk is the same."""
    row = torch.full((vocab,), -float("inf"))
    for i, v in allowed.items():
        row[i] = v
    for given in PARAMETERS:
        u = both_sides(row[:3200], **given)
        check(row.to(dtype).repeat(len(u), 1), u, **given)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3200, 40000])
def test_masks_in_every_chunk(vocab, dtype):
    """Of every four neighbours one is masked, one has the largest value, the others anything below it: tens of thousands of values beyond where bins end."""
    g = torch.Generator().manual_seed(vocab)
    row = 4 - 12 * torch.rand(vocab, generator=g)
    row[::4], row[2::4] = 4.0, -float("inf")
    u = torch.rand(6, generator=g).tolist()
    for given in (dict(), dict(top_p=0.9), dict(top_p=0.9999), dict(min_p=0.01), dict(top_k=vocab // 2), dict(top_k=1024), dict(temperature=2.5, top_p=0.98)):
        check(row.to(dtype).repeat(6, 1), u, **given)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e37, 1e38, 3e38, float("inf")])
def test_finite_logits_farther_apart_than_the_largest_number(temperature, dtype):
    """3e38 and -3e38: the difference is no float32, and the weight is exp(-6e38 / temperature)."""
    inf = float("inf")
    row = torch.full((3200,), -inf)
    row[9], row[20], row[30], row[31] = -3.0e38, 3.0e38, 0.0, -inf
    u = [0.05, 0.1, 0.3, 0.4, 0.6, 0.7, 0.97]
    for vocab in (3200, 40000):
        x = torch.cat([row, torch.full((vocab - 3200,), -inf)]).to(dtype).repeat(len(u), 1)
        for given in (dict(), dict(top_p=0.9), dict(top_k=2), dict(top_k=1500), dict(min_p=0.3)):
            check(x, u, temperature=temperature, **given)
    g = torch.Generator().manual_seed(9)
    x = ((torch.rand(5, 3000, generator=g) * 2 - 1) * 3.3e38).to(dtype)
    for given in (dict(), dict(top_p=0.8), dict(top_k=1200), dict(top_k=30, top_p=0.7)):
        check(x, [0.03, 0.2, 0.47, 0.8, 0.99], temperature=temperature, **given)


def test_the_share_of_a_far_logit():
    """By hand: exp(-2) / (1 + exp(-2)) = 0.119 at a temperature of 3e38, one half without end."""
    x = torch.full((4, 300), -float("inf"))
    x[:, 9], x[:, 20] = -3.0e38, 3.0e38
    assert sampled(x, [0.05, 0.11, 0.13, 0.4], temperature=3e38) == [9, 9, 20, 20]
    assert sampled(x, [0.05, 0.4, 0.49, 0.51], temperature=float("inf")) == [9, 9, 9, 20]


NANS = {torch.float32: (torch.int32, (0x7fc00000, 0x7f800001, 0x7fbfffff, -0x400000, -0x7fffff)), torch.float16: (torch.int16, (0x7e00, 0x7c01, 0x7dff, -0x200, -0x3ff)),
        torch.bfloat16: (torch.int16, (0x7fc0, 0x7f81, 0x7fbf, -0x40, -0x7f))}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_nan_of_any_kind_is_never_a_token(vocab, dtype):
    """Quiet and signalling NaN of both signs among the logits, and in a row of few others."""
    x = (torch.randn(4, vocab, generator=torch.Generator().manual_seed(vocab)) * 2).to(dtype)
    holder, codes = NANS[dtype]
    for i, code in enumerate(codes):
        x.view(holder)[:, i::11] = code
    x.view(holder)[3, 100:] = codes[1]
    assert int(x[:3].isnan().sum()) == 3 * sum(len(range(i, vocab, 11)) for i in range(5)) and not torch.isfinite(x[3, 100:]).any()
    u = [0.02, 0.35, 0.66, 0.97]
    for given in (dict(), dict(top_p=0.9), dict(top_k=20), dict(min_p=0.05), dict(temperature=0.0)):
        check(x, u, **given)
    # the largest beside signalling ones in its 16 bytes, at each of their places
    for at in range(8):
        row = torch.zeros(2, vocab, dtype=dtype)
        row.view(holder)[:, 8:16] = codes[1]
        row[0, 8 + at] = 3.0
        row[1, 8 + at] = row[1, 8 + (at + 3) % 8] = 3.0
        check(row, [0.5, 0.5], temperature=0.0)
        check(row, [0.004, 0.004])
