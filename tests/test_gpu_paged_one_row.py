"""Rows of one token whose view has any stride between rows: a transposed column is read as it lies."""
import pytest
import torch

from paged_cases import DEV, Cache, queries
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _column(t):
    """t [1, width] as the transpose of a column: strides (1, 1)."""
    view = t.to(DEV).reshape(-1, 1).clone().t()
    assert view.stride() == (1, 1)
    return view


def _odd(t):
    """The same, off 16 bytes."""
    return torch.cat([t.new_zeros(3), t.view(-1)]).to(DEV)[3:].view(-1, 1).t()


@pytest.mark.parametrize("view", [_column, _odd])
def test_one_token(view):
    cache = Cache([40], 2, 128, 16, seed=31)
    args = cache.device()
    q, k, v = (queries(1, n, 128, BF, seed=i) for i, n in enumerate((6, 2, 2)))
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    cos, sin = torch.rand(2, 48, 128, device=DEV).unbind(0)
    want = K.paged_attention_decode_forward(q.to(DEV), *args)
    assert torch.equal(K.paged_attention_decode_forward(view(q), *args), want)
    assert torch.equal(K.paged_attention_prompt_forward(view(q), *args, cu), K.paged_attention_prompt_forward(q.to(DEV), *args, cu))
    pools = [[t.clone() for t in args[:4]] for _ in range(2)]
    a = K.paged_kv_append_forward(q.to(DEV), k.to(DEV), v.to(DEV), *pools[0], *args[4:], cos_table=cos, sin_table=sin, rope_dim=64)
    b = K.paged_kv_append_forward(view(q), view(k), view(v), *pools[1], *args[4:], cu_steps=cu, cos_table=cos, sin_table=sin, rope_dim=64)
    assert torch.equal(a, b)
    for x, y in zip(*pools):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
