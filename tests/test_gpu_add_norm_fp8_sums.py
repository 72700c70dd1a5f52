"""Residual + RMS normalisation + E4M3 codes: codes and scales of exact sums of squares, rows written over in place."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS, QUANT_EPS = 2.0 ** -20, 2.0 ** -13


@pytest.mark.parametrize("pow2,quant_eps", [(True, QUANT_EPS), (False, 11.0)])
def test_codes_that_the_root_is_a_factor_of(pow2, quant_eps):
    """With power-of-two scales, and in blocks below quant_eps, the root is a factor of every code: rows of the eight values over and over whose squares lose the most in a
    float32 sum.  Squares, sum, root and products in 64 bits: below 2^-45 off."""
    rng = np.random.default_rng(0)
    eight = rng.standard_normal((200000, 8)).astype(np.float16).astype(np.float64)
    part = np.zeros(len(eight), dtype=np.float32)
    for i in range(8):
        part = (part.astype(np.float64) + eight[:, i] ** 2).astype(np.float32)
    worst = np.argsort(-np.abs(part / (eight ** 2).sum(1) - 1))[:512]
    rng = np.random.default_rng(1)
    x = np.tile(eight[worst], (1, 1024)) * np.where(rng.random((512, 8192)) < 0.5, -1, 1)
    w = (1 + 0.2 * rng.standard_normal(8192)).astype(np.float32)
    codes, scales, _ = K.fused_add_rms_norm_fp8_forward(torch.from_numpy(x).half().to(DEV), None, torch.from_numpy(w).to(DEV), EPS, quant_eps=quant_eps, round_scale_pow2=pow2)
    n, s = P.add_norm(x, w, EPS, quant_eps, pow2)
    assert (np.abs(scales.cpu().numpy() - s) <= (0.0 if pow2 else 2.0 ** -23) * s).all()
    v = n / np.repeat(s, 128, axis=1)
    got, lo, hi = codes.cpu().float().numpy().astype(np.float64), P.e4m3_round(v - np.abs(v) * 2.0 ** -45), P.e4m3_round(v + np.abs(v) * 2.0 ** -45)
    assert ((got >= lo) & (got <= hi)).all(), f"{((got < lo) | (got > hi)).sum()} codes are another value's"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [128, 640, 5120, 8320])
@pytest.mark.parametrize("onto", ["residual", "x"])
def test_in_place_where_the_first_sums_are_zeros(dim, dtype, onto):
    """Lanes behind the row's end neither read what others write over nor say how the row is summed: equal bits, whatever its first eight sums are."""
    g = torch.Generator().manual_seed(dim)
    x, r = torch.randn(64, dim, generator=g).to(dtype), torch.randn(64, dim, generator=g).to(dtype)
    x[:, :8], r[:, :8] = 1, -1
    r[32:, :8] = 1
    x, r, w = x.to(DEV), r.to(DEV), torch.ones(dim, device=DEV)
    want = K.fused_add_rms_norm_fp8_forward(x, r, w, EPS)
    for _ in range(5):
        a, b = (x.clone(), r.clone())
        if onto == "x":
            a, b = b, a                                                       # (the sum is the same)
        got = K.fused_add_rms_norm_fp8_forward(a, b, w, EPS, in_place=True)
        assert got[2].data_ptr() == b.data_ptr()
        for y, z in zip(got, want):
            assert torch.equal(y.view(torch.uint8), z.view(torch.uint8))
