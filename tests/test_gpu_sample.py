"""sample_tokens_forward against its float64 form, token for token.  Random logits and numbers keep away from borders: a weight is rounded to 2^-44 of the largest one, so
the sums of n of them are off by n 2^-44 at most (as an absolute number: their total is 1 or more), and a token can differ only where the form's own nearest border is closer
than that; the tests ask for it to be farther and would say so."""
import numpy as np
import pytest
import torch

from oracle import tree_oracle as T
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(logits, uniform, **given):
    """given: numbers, or lists of a number per row."""
    rows = logits.size(0)
    dtypes = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    args = {n: torch.tensor(v, dtype=dtypes[n], device=DEV) if isinstance(v, list) else v for n, v in given.items()}
    got = K.sample_tokens_forward(logits.to(DEV), torch.tensor(uniform, dtype=torch.float32, device=DEV), **args)
    torch.cuda.synchronize()
    assert got.dtype == torch.int64 and got.shape == (rows,)
    got, x, u = got.tolist(), logits.double().cpu().numpy(), np.array(uniform, dtype=np.float32).astype(np.float64)
    for r in range(rows):
        row = {n: (v[r] if isinstance(v, list) else v) for n, v in given.items()}
        row = {n: int(v) if n == "top_k" else float(np.float32(v)) for n, v in row.items()}
        want, near = T.sample(x[r], u[r], **row)
        assert near > 1, "the case sits on a border"
        assert got[r] == want, (r, got[r], want, row)


def uniforms(n, seed=0):
    return np.random.default_rng(seed).random(n).astype(np.float32).tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,spread", [(1, 1, 1.0), (3, 7, 2.0), (9, 640, 3.0), (64, 1000, 1.0), (5, 4099, 5.0), (4, 32000, 2.0), (2, 200064, 2.0)])
def test_random_rows(rows, vocab, spread, dtype):
    logits = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)) * spread).to(dtype)
    pick = lambda *v: [v[(r * 7 + vocab) % len(v)] for r in range(rows)]
    u = uniforms(rows, rows)
    check(logits, u)
    check(logits, u, temperature=0.7, top_k=40, top_p=0.9, min_p=0.02)
    check(logits, u, temperature=pick(1.0, 0.0, 0.2, 3.0, 40.0), top_k=pick(0, 5, 1, 100, 3000), top_p=pick(1.0, 0.5, 0.95, 0.1), min_p=pick(0.0, 0.3, 0.001))
    check(logits, u, top_p=0.99)
    check(logits, u, top_k=max(1, vocab // 2), temperature=2.0)


def test_every_share_of_a_small_row():
    """A row once for each of many numbers: every token as often as its share."""
    x = torch.tensor([0.3, 2.0, -1.0, 2.0, 0.0, 1.5, float("-inf"), float("nan")])
    n = 500
    check(x.repeat(n, 1), ((np.arange(n) + 0.37) / n).tolist(), top_k=5, temperature=0.9)
    check(x.repeat(n, 1), ((np.arange(n) + 0.37) / n).tolist(), top_p=0.8)


def sampled(logits, uniform, **given):
    return K.sample_tokens_forward(logits.to(DEV), torch.tensor(uniform, dtype=torch.float32, device=DEV), **given).tolist()


@pytest.mark.parametrize("vocab", [8, 5000, 100000])
def test_equal_logits_go_by_their_index(vocab):
    """Sums of equal weights are whole numbers: on the borders too the token is what the definition says.  5000 and more equal ones are cut without a list."""
    x = torch.full((6, vocab), 1.25)
    half = vocab // 2
    u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0]
    whole = [int(v * vocab) for v in u[:4]] + [vocab - 1] * 2
    assert sampled(x, u) == whole
    first = [int(v * half) for v in u[:4]] + [half - 1] * 2
    assert sampled(x, u, top_k=half) == first
    assert sampled(x, u, top_p=0.5) == first
    assert sampled(x, u, top_k=half, top_p=0.5) == [int(v * (half // 2)) for v in u[:4]] + [half // 2 - 1] * 2
    assert sampled(x, u, min_p=1.0) == whole
    # two levels: the cut inside the lower one
    x[:, 3] = 2.0
    assert sampled(x, [0.0] * 6, top_k=1) == [3] * 6 and sampled(x, [0.0] * 6, temperature=0.0) == [3] * 6
    if vocab > 8:
        got = sampled(x, [1.0] * 6, top_k=half)                              # the largest and the first half - 1 others
        assert got == [half - 1] * 6


def test_many_equal_logits_at_the_cut():
    """More equal values at a cut than the list holds, beside others above and below them."""
    vocab, level = 30000, 20000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, vocab, generator=g)
    x[:, torch.randperm(vocab, generator=g)[:level]] = 0.5
    check(x, [0.11, 0.52, 0.93], top_p=0.7)
    check(x, [0.11, 0.52, 0.93], top_k=15000)
    check(x, [0.13, 0.57, 0.91], top_k=15000, top_p=0.83, temperature=[0.5, 1.0, 2.0])


def test_masked_infinite_and_nan_logits():
    inf, nan = float("inf"), float("nan")
    x = torch.full((8, 300), -inf)
    x[1, 7] = 0.0                                                             # one token left
    x[2] = nan
    x[3, 5], x[3, 9], x[3, 20] = nan, -3.0e38, 3.0e38
    x[4, 8], x[4, 100], x[4, 101] = inf, inf, 5.0                             # of infinite ones each has the same share
    x[5] = torch.finfo(torch.float32).min                                     # masks of the type's lowest value: all the same
    x[6, :2] = torch.tensor([-0.0, 0.0])                                      # equal
    x[7, 33] = -3.4e38
    for t in (1.0, 1e-30, 3e38, inf):
        assert sampled(x, [0.5] * 8, temperature=t) == [-1, 7, -1, 20 if t < 1e38 else (9, 20)[1], 100, 150, 1, 33]
    assert sampled(x, [0.4] * 8, temperature=0.0) == [-1, 7, -1, 20, 8, 0, 0, 33]
    for given in (dict(top_k=3), dict(top_p=0.9), dict(top_p=0.0), dict(min_p=1.0), dict(top_k=2, top_p=0.99, min_p=0.5)):
        got = sampled(x, [0.0] * 8, **given)
        assert got == [-1, 7, -1, 20, 8, 0, 0, 33]


def test_numbers_and_parameters_outside_their_ranges():
    x = torch.randn(7, 400, generator=torch.Generator().manual_seed(1))
    first, last = sampled(x, [0.0] * 7), sampled(x, [1.0] * 7)
    assert sampled(x, [-1.0, float("nan"), -float("inf"), -1e-30, -0.0, 0.0, -5.0]) == first and sampled(x, [1.0, 2.0, float("inf"), 1e30, 1.5, 1.0, 7.0]) == last
    best = x.argmax(-1).tolist()
    column = lambda v, dtype=torch.float32: torch.full((7,), v, dtype=dtype, device=DEV)
    assert sampled(x, [0.6] * 7, temperature=column(-1.0)) == best and sampled(x, [0.6] * 7, temperature=column(float("nan"))) == best
    whole = sampled(x, [0.6] * 7)
    assert sampled(x, [0.6] * 7, top_k=column(-4, torch.int32)) == whole and sampled(x, [0.6] * 7, top_k=column(2**31 - 1, torch.int32)) == whole
    assert sampled(x, [0.6] * 7, top_p=column(float("nan"))) == whole and sampled(x, [0.6] * 7, top_p=2.0) == whole and sampled(x, [0.6] * 7, top_k=10**12) == whole
    assert sampled(x, [0.6] * 7, top_p=column(-2.0)) == best and sampled(x, [0.6] * 7, min_p=column(9.0)) == best and sampled(x, [0.6] * 7, min_p=column(float("nan"))) == whole


def test_strides_slices_and_single_values():
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(5, 1013, generator=g).to(dtype).to(DEV)
        u = torch.tensor(uniforms(5), device=DEV)
        for lo, hi in ((0, 1000), (1, 1000), (3, 996), (7, 8), (500, 1013)):
            part = wide[:, lo:hi]
            want = K.sample_tokens_forward(part.contiguous(), u, top_k=30, top_p=0.9)
            assert torch.equal(K.sample_tokens_forward(part, u, top_k=30, top_p=0.9), want)
            assert torch.equal(K.sample_tokens_forward(part[2:3], u[2:3], top_k=30, top_p=0.9), want[2:3])
        turned = wide[:, :64].t()                                              # columns: copied
        assert torch.equal(K.sample_tokens_forward(turned, torch.rand(64, device=DEV) * 0 + 0.3), K.sample_tokens_forward(turned.contiguous(), torch.full((64,), 0.3, device=DEV)))
    assert K.sample_tokens_forward(torch.empty(0, 9, device=DEV), torch.empty(0, device=DEV)).shape == (0,)


def test_a_row_does_not_depend_on_its_batch():
    x = (torch.randn(300, 50000, generator=torch.Generator().manual_seed(4)) * 2).to(torch.bfloat16).to(DEV)
    u = torch.tensor(uniforms(300, 4), device=DEV)
    for given in (dict(), dict(top_k=50, top_p=0.95), dict(top_p=0.99, temperature=1.5)):
        every = K.sample_tokens_forward(x, u, **given)
        for r in (0, 123, 299):
            assert K.sample_tokens_forward(x[r:r + 1], u[r:r + 1], **given).item() == every[r].item()
        assert torch.equal(K.sample_tokens_forward(x, u, **given), every)


def test_the_largest_vocabulary():
    vocab = 2 ** 20
    x = torch.randn(1, vocab, generator=torch.Generator().manual_seed(5)) * 2
    check(x, [0.61], top_p=0.9, temperature=1.3)
    assert sampled(torch.zeros(1, vocab), [0.75]) == [3 * vocab // 4] and sampled(torch.zeros(1, vocab), [0.5], top_k=vocab // 2) == [vocab // 4]


def test_captured_and_replayed_on_two_streams():
    rows, vocab = 6, 9000
    x, u = torch.randn(rows, vocab, device=DEV), torch.rand(rows, device=DEV)
    t, k = torch.full((rows,), 0.8, device=DEV), torch.full((rows,), 50, dtype=torch.int32, device=DEV)
    call = lambda: K.sample_tokens_forward(x, u, temperature=t, top_k=k, top_p=0.95)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = call()
    g = torch.Generator(device=DEV).manual_seed(6)
    for i in range(4):
        x.copy_(torch.randn(rows, vocab, generator=g, device=DEV) * (1 + i))
        u.copy_(torch.rand(rows, generator=g, device=DEV))
        k.fill_([3, 0, 4000, 1][i])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("count", [60, 65, 300, 512, 513, 1500, 2049])
def test_cuts_inside_equal_logits(count, apart, dtype):
    """So many equal values at a cut, one beside the other or all over the row, some of them kept."""
    vocab, g = 20000, torch.Generator().manual_seed(count)
    for rows, wide in ((3, vocab), (3, 3200)):                                # in slices; a workgroup per row
        x = (torch.randn(rows, wide, generator=g) * 0.3 - 4).to(dtype)
        x[:, wide // 2:wide // 2 + 20] = (torch.rand(20, generator=g) + 1).to(dtype)
        at = torch.randperm(wide // 2, generator=g)[:count] if apart else torch.arange(100, 100 + count)
        if count > wide // 2 - 100:
            continue
        x[:, at] = 0.25
        u = uniforms(rows, count)
        keep = 20 + count // 3
        check(x, u, top_k=keep)
        check(x, u, top_k=keep, top_p=0.77)
        # what the 20 and a third of the equal ones have of everything, between two of them
        w = np.exp(x[0].double().numpy() - x[0].double().max().item())
        level = np.exp(0.25 - x[0].double().max().item())
        share = (w[x[0].double().numpy() > 0.25].sum() + (keep - 20 + 0.4) * level) / w.sum()
        check(x[:1].repeat(rows, 1), u, top_p=float(share))


@pytest.mark.parametrize("count,levels", [(90, 5), (400, 7), (500, 16), (700, 5)])
def test_cuts_among_neighbouring_floats(count, levels):
    """Values that differ by single steps of a float32, more of them in one part of a bin than are compared one with another, and more than are ordered."""
    vocab, g = 9000, torch.Generator().manual_seed(count)
    x = torch.rand(2, vocab, generator=g) * 4 - 30
    x[:, :3] = torch.tensor([0.0, -0.5, -1.0])
    near = torch.tensor(-5.0)
    steps = near + torch.arange(levels) * 2.0 ** -21                          # (a step of float32 from 4 to 8)
    at = torch.randperm(vocab - 3, generator=g)[:count] + 3
    x[:, at] = steps[torch.randint(levels, (count,), generator=g)]
    u = uniforms(2, count)
    w = np.exp(x[0].double().numpy())
    check(x[:1].repeat(2, 1), u, top_p=float((w[:3].sum() + (count // 2 + 0.4) * np.exp(-5.0)) / w.sum()))
    check(x, u, top_k=3 + count // 2)
    check(x, u, top_k=3 + count // 2, top_p=0.9, temperature=1.5)


def test_more_rows_than_compute_units_with_parameters_of_their_own():
    """Long rows of mixed parameters are taken in another order than they stand in; more of them than that is done for are not."""
    g = torch.Generator().manual_seed(8)
    rows, vocab = 270, 9000
    x = (torch.randn(rows, vocab, generator=g) * 2).to(torch.float16)
    pick = lambda *v: [v[int(i)] for i in torch.randint(len(v), (rows,), generator=g)]
    given = dict(temperature=pick(0.0, 0.5, 1.0, 2.0, -1.0), top_k=pick(0, 1, 30, 1000, 2000, -3), top_p=pick(1.0, 0.9, 0.5), min_p=pick(0.0, 0.05))
    check(x, uniforms(rows, 9), **given)
    check(x, uniforms(rows, 9), top_k=given["top_k"])
    big = 4100
    x = (torch.randn(big, vocab, generator=g) * 2).to(torch.bfloat16).to(DEV)
    u = torch.tensor(uniforms(big, 10), device=DEV)
    k = torch.randint(0, 3, (big,), generator=g).int().to(DEV) * 20
    t = torch.randint(0, 3, (big,), generator=g).float().to(DEV)
    whole = K.sample_tokens_forward(x, u, temperature=t, top_k=k, top_p=0.95)
    for n in (4096, 1000, 300):
        parts = [K.sample_tokens_forward(x[i:i + n], u[i:i + n], temperature=t[i:i + n], top_k=k[i:i + n], top_p=0.95) for i in range(0, big, n)]
        assert torch.equal(torch.cat(parts), whole)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [4000, 30000])
def test_cuts_inside_a_crowd(vocab, dtype):
    """Most values close together far below the largest: more of them in the bin of the cut than the list holds, different ones and (in fp16) equal ones too."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(4, vocab, generator=g) * 0.003 - 6
    x[:, 17], x[:, 40], x[:, 41] = 0.0, -1.0, -35.0
    x = x.to(dtype)
    u = uniforms(4, vocab)
    check(x, u, top_p=0.99)
    check(x, u, top_p=[0.5, 0.9, 0.97, 0.995], min_p=0.0005)
    check(x, u, top_p=0.98, temperature=2.0, top_k=vocab - 1)
    check(x, u, top_p=0.9, top_k=vocab // 2 + 500)
