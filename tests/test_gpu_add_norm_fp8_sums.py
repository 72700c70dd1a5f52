"""Residual + RMS normalisation + E4M3 codes: rows written over in place."""
import pytest
import torch

from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 2.0 ** -20


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
