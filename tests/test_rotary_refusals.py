"""Refusals of the norms with rotation that come before any launch, without a GPU: tensors
in host memory that say they are on one, which nothing may read."""

import pytest
import torch

from pipeswift_amd import rotary


class OnGpu(torch.Tensor):
    @property
    def is_cuda(self):
        return True


def _gpu(t):
    return t.as_subclass(OnGpu)


def _inputs(P=500, rot=64):
    N, H, D = 4, 2, 64
    zeros = lambda *shape, dtype=torch.bfloat16: _gpu(torch.zeros(*shape, dtype=dtype))  # noqa: E731
    return dict(q=zeros(N, 4, D), k=zeros(N, H, D), positions=zeros(N, dtype=torch.int64),
                cos_sin=zeros(P, rot, dtype=torch.float32))


@pytest.mark.parametrize("stride", [0, 1, 63])
def test_tables_whose_rows_overlap(stride):
    """A broadcast table, or rows closer than they are long."""
    x = _inputs()
    x["cos_sin"] = _gpu(torch.zeros(500 * 64).as_strided((500, 64), (stride, 1)))
    with pytest.raises(AssertionError, match="cos_sin"):
        rotary.norm_rope(**x)
