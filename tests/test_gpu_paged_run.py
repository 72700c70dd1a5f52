"""The paged operators one after the other, as a server runs them: norm with codes, product with FP8 weights, append, attention, the next norm.  Prompts, then
prompts and single tokens in one batch, then decode steps from a captured graph.  Every operator is held to its float64 form on what the one before it gave."""
import numpy as np
import pytest
import torch

from paged_cases import DEV, Cache, close
from pocketllm_amd import hip_kernel as K
from test_gpu_add_norm_fp8 import EPS, _check_codes
from test_gpu_paged_append import _check as check_append
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV_HEADS, DIM, ROPE = 512, 12, 2, 64, 32
WIDTH, KV_WIDTH = HEADS * DIM, KV_HEADS * DIM


class Layer:
    def __init__(self, positions):
        g = torch.Generator().manual_seed(0)
        weights = [(torch.randn(n, k, generator=g) * 40).to(torch.float8_e4m3fn) for n, k in ((WIDTH + 2 * KV_WIDTH, HIDDEN), (HIDDEN, WIDTH))]
        self.qkv, self.out = [(w.to(DEV), torch.full((w.size(0) // 128, w.size(1) // 128), 1e-3, device=DEV)) for w in weights]
        self.norm = (1.0 + 0.1 * torch.randn(HIDDEN, generator=g)).to(DEV)
        self.tables = P.rotary_rows(positions, DIM, ROPE)
        self.cos, self.sin = (torch.from_numpy(t).to(DEV) for t in self.tables)

    def __call__(self, x, stream, cache, cu=None, note=None):
        """(what goes to the next norm as x, the residual stream); `note` gets what lies between."""
        codes, scales, stream = K.fused_add_rms_norm_fp8_forward(x, stream, self.norm, EPS)
        rows = K.fp8_gemm_forward(codes, scales, *self.qkv, out_dtype=x.dtype)
        q, k, v = rows.split([WIDTH, KV_WIDTH, KV_WIDTH], dim=-1)
        turned = K.paged_kv_append_forward(q, k, v, *cache, cu_steps=cu, cos_table=self.cos, sin_table=self.sin, rope_dim=ROPE)
        mixed = K.paged_attention_decode_forward(turned, *cache) if cu is None else K.paged_attention_prompt_forward(turned, *cache, cu)
        if note is not None:
            note.update(codes=codes, scales=scales, stream=stream, q=q, k=k, v=v, turned=turned, mixed=mixed)
        codes, scales = K.fp8_act_quant_forward(mixed)
        return K.fp8_gemm_forward(codes, scales, *self.out, out_dtype=x.dtype), stream


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,width", [(32, 12), (64, 17)])                   # tables of less and of more than one run
def test_prompts_mixed_batches_and_decode_steps(page, width, dtype):
    layer, seqs = Layer(page * width), 3
    shape = Cache([page * width] * seqs, KV_HEADS, DIM, page, seed=page, width=width)
    shape.key_codes[:], shape.value_codes[:] = 0x7f, 0xff                      # pages in no order, nothing in them yet
    shape.key_scales[:], shape.value_scales[:] = np.nan, np.nan
    cache = list(shape.device())
    held, g = np.zeros(seqs, dtype=np.int32), torch.Generator().manual_seed(7)

    def some(tokens):
        return tuple((torch.randn(tokens, HIDDEN, generator=g) * s).to(dtype).to(DEV) for s in (1.0, 3.0))

    for steps in ([70, 1, 133], [1, 90, 0], [1, 1, 1]):
        held += np.array(steps, dtype=np.int32)
        cache[5].copy_(torch.from_numpy(held))
        cu, note = np.concatenate([[0], np.cumsum(steps)]), {}
        x, stream = some(cu[-1])
        before = [t.view(torch.uint8).cpu().numpy().copy() for t in cache[:2]] + [t.cpu().numpy().copy() for t in cache[2:4]]
        even = steps == [1, 1, 1]
        y, _ = layer(x, stream, cache, None if even else torch.tensor(cu, dtype=torch.int32, device=DEV), note)
        torch.cuda.synchronize()
        assert torch.equal(note["stream"], (x.float() + stream.float()).to(dtype)) and bool(torch.isfinite(y).all())
        _check_codes(note["codes"], note["scales"], note["stream"], layer.norm, False)
        shape.lengths = held.copy()
        check_append(shape, before, cache, note["turned"], *(note[n].cpu() for n in "qkv"), cu, ROPE, *layer.tables, HEADS)
        shape.key_codes, shape.value_codes = (t.view(torch.uint8).cpu().numpy() for t in cache[:2])
        shape.key_scales, shape.value_scales = (t.cpu().numpy() for t in cache[2:4])
        turned = note["turned"].cpu()
        close(note["mixed"], *shape.attention(turned.double().numpy().reshape(-1, HEADS, DIM), cu), dtype)

    # decode steps of a graph that moves the lengths on itself, against the same steps one by one on a copy of the cache
    x, stream = some(seqs)
    copy = [t.clone() for t in cache]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, stream, [t.clone() for t in cache])                           # (workspaces and code, before the capture)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        cache[5].add_(1)
        kept = layer(x, stream, cache)
    for _ in range(3):
        x2, stream2 = some(seqs)
        x.copy_(x2)
        stream.copy_(stream2)
        graph.replay()
        copy[5].add_(1)
        want = layer(x2, stream2, copy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, copy))
