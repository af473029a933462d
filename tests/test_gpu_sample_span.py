"""Rows whose largest and smallest logits are further apart than the type's largest value: which tokens are among the first k
does not depend on the difference, and at temperatures of that size, up to infinity, all of them weigh something."""
import math

import pytest
import torch
from test_gpu_sample import check
from test_gpu_top_logits import check as check_top

pytestmark = pytest.mark.gpu


def _x(dev, V, dtype):
    high = torch.finfo(dtype).max
    i = torch.arange(V, device=dev)
    g = torch.Generator(device=dev).manual_seed(V)
    n = torch.rand(V, generator=g, device=dev) * 2 - 1
    rows = [torch.where(i % 97 == 5, high, -high), torch.where(i == 3, 3e38, -3e38), n * high, torch.where(n > 0.9, n * high, -high),
            torch.where(i % 2 == 0, -high, torch.where(i == 31, 2e38, -math.inf)), torch.where(i == 8, high, n - 3e38)]
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,ks", [(100, (1, 50, 99)), (4001, (20, 100, 400, 900, 2000)), (70003, (50, 1000))])
def test_draws(cuda_device, dtype, V, ks):
    x = _x(cuda_device, V, dtype)
    u = torch.tensor([0.03, 0.31, 0.48, 0.66, 0.85, 0.97], device=cuda_device)
    for k in ks:
        for T in (1.0, 1e38, math.inf):
            check(x, u, {"temperature": T, "top_k": k}, edges=False)
            check(x, u, {"temperature": T, "top_k": k, "top_p": 0.7, "min_p": 0.01}, edges=False)
    if V < 10000:
        for copies in (50, 100):  # with 512 and with 256 threads to a row
            check(x.repeat(copies, 1), u.repeat(copies), {"temperature": math.inf, "top_k": ks[1]}, edges=False)
        each = {"temperature": torch.tensor([1e38, math.inf] * 3, device=cuda_device),
                "top_k": torch.full((6,), ks[1], dtype=torch.int32, device=cuda_device)}
        check(x, u, each, edges=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_logits(cuda_device, dtype):
    for V, ks in ((100, (1, 50, 99)), (4001, (20, 100, 400, 1000)), (70003, (50, 1000))):
        x = _x(cuda_device, V, dtype)
        for k in ks:
            check_top(x, k, 1.0)
            check_top(x.repeat(100, 1), k, 1.0)
