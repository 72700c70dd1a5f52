"""Caches for the tests of the paged E4M3 operators: pages in no order, unused slots and pages full of NaN codes and NaN scales, table entries behind a
sequence's last page that lie outside the pool."""
import numpy as np
import torch

from oracle import paged_oracle as P

DEV = "cuda:0"


class Cache:
    """Host copies (numpy) and device tensors of a pool, its table and lengths."""

    def __init__(self, lengths, kv_heads, dim, page, seed=0, spare=3, width=None, scale_exponents=(-8, -4)):
        rng = np.random.default_rng(seed)
        counts = [-(-max(n, 0) // page) for n in lengths]
        pool, width = sum(counts) + spare, width or max(max(counts), 1)
        self.kv_heads, self.dim, self.page, self.pool, self.width = kv_heads, dim, page, pool, width
        self.lengths = np.array(lengths, dtype=np.int32)
        self.table = np.full((len(lengths), width), pool + 5, dtype=np.int32)
        self.key_codes = np.full((pool, kv_heads, page, dim), 0x7f, dtype=np.uint8)
        self.value_codes = np.full((pool, kv_heads, dim, page), 0xff, dtype=np.uint8)
        self.key_scales = np.full((pool, kv_heads), np.nan, dtype=np.float32)
        self.value_scales = np.full((pool, kv_heads), np.nan, dtype=np.float32)
        order, at = rng.permutation(pool - 1) + 1, 0                           # (page 0 is never used: its scales stay NaN)
        for s, c in enumerate(counts):
            for p in range(c):
                which = order[at]
                at += 1
                self.table[s, p] = which
                n = min(page, lengths[s] - p * page)
                self.key_codes[which, :, :n] = self._codes(rng, kv_heads, n, dim)
                self.value_codes[which, :, :, :n] = self._codes(rng, kv_heads, dim, n)
                self.key_scales[which] = 2.0 ** rng.integers(*scale_exponents, kv_heads)
                self.value_scales[which] = 2.0 ** rng.integers(*scale_exponents, kv_heads)

    @staticmethod
    def _codes(rng, *shape):
        v = torch.from_numpy(np.clip(rng.standard_normal(shape) * 60, -448, 448)).float()
        return v.to(torch.float8_e4m3fn).view(torch.uint8).numpy()

    def device(self):
        """The tensors that the operators take, in their order."""
        f8 = torch.float8_e4m3fn
        return (torch.from_numpy(self.key_codes).to(DEV).view(f8), torch.from_numpy(self.value_codes).to(DEV).view(f8), torch.from_numpy(self.key_scales).to(DEV),
                torch.from_numpy(self.value_scales).to(DEV), torch.from_numpy(self.table).to(DEV), torch.from_numpy(self.lengths).to(DEV))

    def attention(self, q, cu_steps, scale=None):
        """float64 outputs and their errors' measures for q [tokens, heads, dim]."""
        return P.attention(q, self.key_codes, self.value_codes, self.key_scales, self.value_scales, self.table, self.lengths, cu_steps,
                           self.dim ** -0.5 if scale is None else scale)


def queries(tokens, heads, dim, dtype, seed=0, size=1.0):
    return (torch.randn(tokens, heads * dim, generator=torch.Generator().manual_seed(seed)) * size).to(dtype)


def close(got, want, note, dtype):
    """Every output within what its roundings can add up to.

    u = half a step of the type.  Softmax weights are rounded to the type once, above the division (u of the weighted mean of |v|) and below it (u of
    the output), the output once (u of itself).  A
    score is a float32 sum of dim exact products (matrix instructions add four or more at a time: below dim + 8 roundings of 2^-24 of the sum of
    magnitudes), scaled twice and turned to base 2 (4 roundings); as an exponent its error is one of the weight.  exp2, the running maximum's and the runs'
    factors: 16 units; the sums of weights and of products: below (keys / 16 + 64) roundings one after the other.  Weights and their error appear above and
    below the division: twice.  fp16 weights below 2^-14 and halved values lose up to 2^-25 each."""
    u = torch.finfo(dtype).eps / 2
    f32 = (note["score"] * (note["spread"].shape[-1] + 12) + 16 + note["keys"] / 16 + 64) * 2.0 ** -24
    bound = u * (note["spread"] + 2 * np.abs(want)) * (1 + 3 * u) + 2 * f32 * (note["spread"] + np.abs(want))
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (note["keys"] * note["top"] + 4)
    got = got.detach().cpu().double().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
    ok = np.isnan(want) | (np.abs(got - want) <= bound)
    assert ok.all(), f"{(~ok).sum()} outputs off, the worst by {np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)):.2f} bounds"
