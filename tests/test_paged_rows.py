"""Rows as the paged operators read them, without a GPU: the stride of a single row is the row's width, whatever its view says."""
import pytest
import torch

from pocketllm_amd import hip_kernel as K


@pytest.mark.parametrize("start", [0, 3])
def test_the_stride_of_one_row(start):
    flat = torch.arange(131, dtype=torch.bfloat16)[start:start + 128]
    for t in (flat.view(-1, 1).t(), flat.view(1, -1), flat.view(-1, 1).t()[:, :64], torch.zeros(128, 5, dtype=torch.bfloat16)[:, :1].t()):
        rows = K._rows16(t)
        assert rows.stride() == (t.size(1), 1) and rows.data_ptr() % 16 == 0 and torch.equal(rows, t)


def test_rows_that_the_kernels_read_as_they_lie():
    wide = torch.zeros(4, 192, dtype=torch.float16)
    for t in (wide[:, :128], wide[:, 64:], wide[::2, :64], wide[:1, :128]):
        rows = K._rows16(t)
        assert rows.data_ptr() == t.data_ptr() and (t.size(0) == 1 or rows.stride() == t.stride())
    for t in (wide[:, 3:131], wide[:1].expand(4, 192), wide.t()):
        rows = K._rows16(t)
        assert rows.is_contiguous() and rows.data_ptr() % 16 == 0 and torch.equal(rows, t)
