"""Rows with fewer pieces of 8 than logits that are asked for, or hardly more: no bound comes from the pieces' maxima, and what
is gathered is the whole row, or more than there is room for."""
import pytest
import torch
from test_gpu_sample import check as check_draw
from test_gpu_top_logits import check

pytestmark = pytest.mark.gpu

SIZES = [(3, 3000, 400), (300, 3000, 400), (2, 4096, 600), (300, 4095, 500), (3, 8192, 1000), (3, 8193, 1000), (300, 8193, 500),
         (600, 900, 120), (600, 1000, 125), (600, 511, 64), (600, 513, 65), (2, 2047, 1024), (2, 2049, 1024)]


def _x(dev, rows, V, dtype):
    g = torch.Generator(device=dev).manual_seed(rows + V)
    return (torch.randn(rows, V, generator=g, device=dev) * 3).to(dtype), torch.rand(rows, generator=g, device=dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,k", SIZES)
def test_top_logits(cuda_device, dtype, rows, V, k):
    check(_x(cuda_device, rows, V, dtype)[0], k, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,k", SIZES)
def test_draws(cuda_device, dtype, rows, V, k):
    x, u = _x(cuda_device, rows, V, dtype)
    check_draw(x, u, {"top_k": k, "temperature": 1.3}, edges=False)
