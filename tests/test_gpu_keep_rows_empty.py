"""Entries of tensors that have none: whole rows of zeros."""
import pytest
import torch

from vet_amd import torch_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape, dtype", [((1, 0, 37), torch.float32), ((6, 0, 5, 2), torch.bfloat16), ((2, 0, 64), torch.uint8), ((2, 0), torch.int64), ((3, 0, 0), torch.float32)])
def test_rows_of_a_tensor_without_entries(shape, dtype, rasterizer):
    index = torch.arange(50, device="cuda", dtype=torch.int32).expand(shape[0], 50).contiguous()
    x = torch.empty(shape, dtype=dtype, device="cuda")
    full = torch.empty((shape[0], 50) + shape[2:], dtype=dtype, device="cuda")
    if full.numel():
        full.view(torch.uint8).fill_(0xFF)  # what the result's memory held before
    del full
    (got,) = rasterizer.keep_rows([x], index)
    assert got.shape == (shape[0], 50) + shape[2:] and not got.any()
    (same,) = torch_ops.keep_rows([x], index, [1])
    assert same.shape == got.shape and not same.any()


def test_no_outers(rasterizer):
    (got,) = rasterizer.keep_rows([torch.empty((0, 4, 3), device="cuda")], torch.zeros((1, 2), dtype=torch.int32, device="cuda"))
    assert got.shape == (0, 2, 3)
