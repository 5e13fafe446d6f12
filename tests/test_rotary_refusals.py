"""Refusals of the norms with rotation that come before any launch, without a GPU: tensors
in host memory that say they are on one, which nothing may read."""

import pytest
import torch

from pipeswift_amd import rotary
from pipeswift_amd._lib import overlap


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


@pytest.mark.parametrize("kind", ["same", "fp8", "mxfp4"])
@pytest.mark.parametrize("name,side", [("q_out", 0), ("q_out", 1), ("k_out", 0), ("k_out", 1)])
def test_outputs_that_lie_in_a_cache(kind, name, side):
    """Where the append writes, whatever the cache's type; beside it they are no concern."""
    x = _inputs()
    heads, D = (4, 64) if name == "q_out" else (2, 64)
    store = torch.zeros(1 << 16, dtype=torch.uint8)
    entry, dtype, size = {"same": (64, torch.bfloat16, 2), "fp8": (64, torch.float8_e4m3fn, 1), "mxfp4": (36, torch.uint8, 1)}[kind]
    fused = store[:3 * 2 * 16 * 2 * entry * size].view(dtype).view(3, 2, 16, 2, entry)
    at = side * 16 * 2 * entry * size  # where that cache begins
    out = store[at:at + 4 * heads * D * 2].view(torch.bfloat16).view(4, heads, D)
    x |= dict(v=_gpu(torch.zeros(4, 2, D, dtype=torch.bfloat16)), key_cache=_gpu(fused[:, 0]), value_cache=_gpu(fused[:, 1]),
              slot_mapping=_gpu(torch.arange(4)))
    with pytest.raises(AssertionError, match=f"{name} must be its input itself or share no element"):
        rotary.norm_rope_and_cache(**x, **{name: _gpu(out)})


def test_columns_side_by_side_do_not_overlap():
    """What is taken for columns beside each other shares no element, and a projection's columns are."""
    g = torch.Generator().manual_seed(1)
    draw = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    store = torch.zeros(4000, dtype=torch.bfloat16)
    found = 0
    for _ in range(3000):
        s, pair = draw(8, 90), []
        for _ in range(2):
            n, heads, dim, gap = draw(1, 5), draw(1, 4), draw(1, 9), draw(0, 20)
            pair.append(store[draw(0, 300):].as_strided((n, heads, dim), (s, gap, 1), store[draw(0, 300):].storage_offset()))
        a, b = pair
        if rotary._side_by_side(a, b):
            found += 1
            assert not overlap(a, b)
    assert found > 300
    q, k, v = torch.zeros(6, 48 * 64).split([32 * 64, 8 * 64, 8 * 64], 1)
    q, k, v = (x.unflatten(1, (-1, 64)) for x in (q, k, v))
    for a in (q, k, v):
        for b in (q, k, v):
            assert rotary._side_by_side(a, b) == (a is not b)
