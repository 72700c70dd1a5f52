"""Residual + RMS normalisation + E4M3 codes in one launch against a float64 form.

Errors counted: the sum of x and residual is rounded once, as torch rounds it (equal bits).  Normalized values: a product of three factors whose
relative error is that of the sum of squares (eight values one after the other in float32, halved by the root): below 8 * 2^-24, held to 2^-18.  Scales inherit
it and one rounding.  Codes round a value that
is off by 2^-17 at most, so each lies between the codes of the two ends."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS, QUANT_EPS = 1e-6, 1e-4


def _inputs(rows, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g).to(dtype)
    r = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)
    w = 1.0 + 0.2 * torch.randn(dim, generator=g)
    return x, r, w


def _check_codes(codes, scales, total, w, pow2):
    codes, scales = codes.cpu().float().numpy().astype(np.float64), scales.cpu().numpy().astype(np.float64)
    n, s = P.add_norm(total.cpu().float().numpy(), w.cpu().numpy(), EPS, QUANT_EPS, pow2)
    if pow2:
        lo, hi = (P.add_norm(total.cpu().float().numpy(), w.cpu().numpy() * f, EPS, QUANT_EPS, True)[1] for f in (1 - 2.0 ** -17, 1 + 2.0 ** -17))
        assert ((scales == lo) | (scales == hi)).all()
    else:
        assert (np.abs(scales - s) <= 2.0 ** -17 * s).all()
    v = n / np.repeat(scales, 128, axis=1)
    lo, hi = P.e4m3_round(v - np.abs(v) * 2.0 ** -16), P.e4m3_round(v + np.abs(v) * 2.0 ** -16)
    assert ((codes >= lo) & (codes <= hi)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,dim,pow2", [(1, 128, False), (1, 5120, False), (3, 384, True), (5, 512, False), (7, 640, True), (4, 2048, False), (3, 2176, True),
                                           (2, 4224, False), (6, 8192, True), (2, 8320, False), (3, 16512, True), (1, 32768, False), (513, 256, False)])
def test_against_float64(rows, dim, pow2, dtype):
    x, r, w = _inputs(rows, dim, dtype, seed=rows + dim)
    codes, scales, total = K.fused_add_rms_norm_fp8_forward(x.to(DEV), r.to(DEV), w.to(DEV), EPS, quant_eps=QUANT_EPS, round_scale_pow2=pow2)
    assert codes.dtype == torch.float8_e4m3fn and scales.shape == (rows, dim // 128)
    assert torch.equal(total.cpu(), (x.float() + r.float()).to(dtype))
    _check_codes(codes, scales, total, w, pow2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_codes_are_those_of_the_exact_values(dtype):
    """Without power-of-two scales the root falls out of a code: 448 t w / max |t w|, a product of 48 bits, a quotient and a product in 64: below 2^-45 off."""
    x, r, w = _inputs(300, 4096, dtype, seed=6)
    codes, _, total = K.fused_add_rms_norm_fp8_forward(x.to(DEV), r.to(DEV), w.to(DEV), EPS, quant_eps=QUANT_EPS)
    n, s = P.add_norm(total.cpu().float().numpy(), w.numpy(), EPS, QUANT_EPS, False)
    v = n / np.repeat(s, 128, axis=1)
    got, lo, hi = codes.cpu().float().numpy().astype(np.float64), P.e4m3_round(v - np.abs(v) * 2.0 ** -45), P.e4m3_round(v + np.abs(v) * 2.0 ** -45)
    assert ((got >= lo) & (got <= hi)).all()


@pytest.mark.parametrize("size", [2.0 ** 90, 2.0 ** -90])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_whose_squares_float32_does_not_hold(dtype, size):
    x, r, w = _inputs(5, 2048, dtype, seed=12)
    x, r = x * size, r * size
    x[3], r[3] = 0, 0
    codes, scales, total = K.fused_add_rms_norm_fp8_forward(x.to(DEV), r.to(DEV), w.to(DEV), 0.0 if size < 1 else EPS, quant_eps=QUANT_EPS)
    live = [0, 1, 2, 4]
    n, s = P.add_norm(total.cpu().float().numpy()[live] / size, w.numpy(), 0.0, QUANT_EPS, False)
    assert (np.abs(scales.cpu().numpy()[live] - s) <= 2.0 ** -17 * s).all()
    v = n / np.repeat(s, 128, axis=1)
    got, lo, hi = codes.cpu().float().numpy().astype(np.float64)[live], P.e4m3_round(v - np.abs(v) * 2.0 ** -45), P.e4m3_round(v + np.abs(v) * 2.0 ** -45)
    assert ((got >= lo) & (got <= hi)).all()
    if size > 1:
        assert (codes[3].float() == 0).all()


def test_in_place_no_residual_and_shapes():
    x, r, w = _inputs(6, 1024, torch.bfloat16)
    xd, rd, wd = x.to(DEV), r.to(DEV), w.to(DEV)
    codes, scales, total = K.fused_add_rms_norm_fp8_forward(xd, rd, wd, EPS)
    stream = rd.clone()
    c2, s2, t2 = K.fused_add_rms_norm_fp8_forward(xd, stream, wd, EPS, in_place=True)
    assert t2.data_ptr() == stream.data_ptr() and torch.equal(stream, total)
    assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2, scales)
    c3, s3, t3 = K.fused_add_rms_norm_fp8_forward(total.view(2, 3, 1024), None, wd, EPS)
    assert t3.data_ptr() == total.data_ptr() and c3.shape == (2, 3, 1024) and s3.shape == (2, 3, 8)
    assert torch.equal(c3.view(torch.uint8).view(6, 1024), codes.view(torch.uint8)) and torch.equal(s3.view(6, 8), scales)
    empty = K.fused_add_rms_norm_fp8_forward(xd[:0], rd[:0], wd, EPS)
    assert [tuple(t.shape) for t in empty] == [(0, 1024), (0, 8), (0, 1024)]


def test_views_that_begin_anywhere_and_columns_of_a_wider_row():
    x, r, w = _inputs(5, 640, torch.float16)
    want = K.fused_add_rms_norm_fp8_forward(x.to(DEV), r.to(DEV), w.to(DEV), EPS)
    wide = torch.zeros(5, 1283, dtype=torch.float16, device=DEV)
    wide[:, 3:643], wide[:, 643:] = x.to(DEV), r.to(DEV)
    flat = torch.zeros(641, device=DEV)
    flat[1:] = w.to(DEV)
    got = K.fused_add_rms_norm_fp8_forward(wide[:, 3:643], wide[:, 643:], flat[1:], EPS)
    for a, b in zip(got, want):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_zeros_infinities_and_nan():
    x = torch.zeros(4, 512, dtype=torch.bfloat16, device=DEV)
    r = torch.ones(4, 512, dtype=torch.bfloat16, device=DEV)
    r[0] = 0
    r[2, 200] = float("inf")
    r[3, 5] = float("nan")
    w = torch.ones(512, device=DEV)
    codes, scales, total = K.fused_add_rms_norm_fp8_forward(x, r, w, EPS, quant_eps=QUANT_EPS)
    assert (codes[0].float() == 0).all() and torch.allclose(scales[0], torch.full((4,), QUANT_EPS / 448, device=DEV))
    assert (codes[1].float() == 448).all()
    # an infinity: its own value is not a number, the rest of the row is divided by an infinite norm
    assert codes[2, 128:256].float().isnan().all() and scales[2, 1].isnan() and (codes[2, :128].float() == 0).all() and (codes[2, 256:].float() == 0).all()
    assert codes[3].float().isnan().all() and scales[3].isnan().all()


def test_feeds_the_fp8_matmul():
    """Codes and scales as fp8_gemm_forward takes them: the product of what they stand for."""
    x, r, w = _inputs(9, 1024, torch.bfloat16, seed=3)
    codes, scales, total = K.fused_add_rms_norm_fp8_forward(x.to(DEV), r.to(DEV), w.to(DEV), EPS)
    weight = (torch.randn(256, 1024, generator=torch.Generator().manual_seed(4)) * 50).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = torch.rand(2, 8, generator=torch.Generator().manual_seed(5)) * 0.01
    y = K.fp8_gemm_forward(codes, scales, weight.to(DEV), ws.to(DEV), out_dtype=torch.float32).cpu().double()
    a = codes.cpu().double() * scales.cpu().double().repeat_interleave(128, 1)
    b = weight.double() * ws.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    want = a @ b.t()
    assert (y - want).norm() <= 1e-3 * want.norm()             # what the framework asks of its matrix products


def test_captured_and_on_another_stream():
    x, r, w = _inputs(33, 5120, torch.bfloat16)
    x, r, w = x.to(DEV), r.to(DEV), w.to(DEV)
    want = [t.clone() for t in K.fused_add_rms_norm_fp8_forward(x, r, w, EPS)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.fused_add_rms_norm_fp8_forward(x, r, w, EPS)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = K.fused_add_rms_norm_fp8_forward(x, r, w, EPS)
    for seed in (1, 2, 3):
        x2, r2, _ = _inputs(33, 5120, torch.bfloat16, seed=seed)
        x.copy_(x2.to(DEV))
        r.copy_(r2.to(DEV))
        graph.replay()
        for a, b in zip(kept, K.fused_add_rms_norm_fp8_forward(x, r, w, EPS)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
