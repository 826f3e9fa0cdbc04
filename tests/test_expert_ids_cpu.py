"""Expert ids of every integer type, as the MXFP4 expert layer takes them."""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

INTEGERS = [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32,
            torch.uint64]


@pytest.mark.parametrize("experts", [4, 16, 128, 200, 512])
@pytest.mark.parametrize("dtype", INTEGERS)
def test_values_are_kept(dtype, experts):
    ids = torch.tensor([[0, 3, 7], [15, 100, 127]]).to(dtype)
    got = ops._expert_ids(ids, experts)
    assert got.dtype is torch.int32 and got.shape == ids.shape
    for a, b in zip(got.flatten().tolist(), [0, 3, 7, 15, 100, 127]):
        assert a == b if b < experts else not 0 <= a < experts


@pytest.mark.parametrize("dtype", INTEGERS)
def test_out_of_range_stays_out(dtype):
    """The types' lowest and highest values, among them ones whose low 32 bits are an expert."""
    f = torch.iinfo(dtype)
    values = [f.min, f.max, f.max - 1]
    if f.bits == 64:
        values += [(1 << 32) + 3, (1 << 40), (1 << 62) + 1]
    experts = 100
    got = ops._expert_ids(torch.tensor(values, dtype=dtype), experts)
    for a, b in zip(got.tolist(), values):
        assert a == b if 0 <= b < experts else not 0 <= a < experts


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.complex64,
                                   torch.bool])
def test_other_types_are_refused(dtype):
    with pytest.raises(TypeError):
        ops._expert_ids(torch.zeros(2, 2).to(dtype), 8)
