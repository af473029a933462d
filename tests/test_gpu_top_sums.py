"""The sums of exponentials behind top_logits' log-sum-exp and top_kl_loss' Z, where their float32 additions would show.

A row holds a 0 in one piece of 8 of each thread and -17.625 everywhere else: 8 exp(-17.625) = 1.487 2^-23, of which an addition
to a sum from 1 to 2 that rounds to 2^-23 keeps 1.  Of a thread's 32 to 128 pieces that would lose 15 to 62 times 2^-23 of the
sum.  The sums carry what an addition rounds off.  Bars, in 2^-24 of the sum: 2 for compensated additions, 3 for the tree over
the piece that holds the 0, 1 for all else of a thread (the small terms, 2.3e-5 of the sum at most, are off by 3 17.625 + 2 times
2^-24 of themselves: 1e-3), and 6 for a wave's float32 sum in the loss; a log-sum-exp takes these as they are, and its own
rounding.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LOW = -17.625


@pytest.mark.parametrize("dtype,rows,V,threads", [(torch.float32, 2, 262144, 1024), (torch.float32, 300, 65536, 512),
                                                  (torch.bfloat16, 2, 262144, 1024), (torch.bfloat16, 300, 131072, 512),
                                                  (torch.bfloat16, 600, 65536, 256)])
def test_log_sum_exp(cuda_device, dtype, rows, V, threads):
    from sparseforge_amd.distill import top_logits

    row = torch.full((V,), LOW, dtype=dtype, device=cuda_device)
    part = V // (threads // 64)  # a wave's
    row.view(-1, part)[:, :512:8] = 0.0
    top = top_logits(row.expand(rows, V), 16, 1.0)
    want = torch.logsumexp(row.double(), 0)
    assert abs(float(want) - math.log(threads)) < 1e-3  # one 0 to a thread
    assert bool(((top.lse.double() - want).abs() <= 2.0 ** -24 * (2 + 3 + 1 + want)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,threads", [(3, 1024), (300, 256)])
@pytest.mark.parametrize("rest", [False, True])
def test_loss(cuda_device, dtype, rows, threads, rest):
    """One listed token at 0 whose teacher is sure of it: the loss is Z; with half of the probability for the rest, it is
    log 1/2 + (Z + Z - Z_rest) / 2."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    V = 262144
    row = torch.full((V,), LOW, dtype=dtype, device=cuda_device)
    row[:threads * 8:8] = 0.0
    ids = torch.zeros(rows, 1, dtype=torch.int32, device=cuda_device)
    values = torch.zeros(rows, 1, dtype=dtype, device=cuda_device)
    if rest:
        lse = torch.full((rows,), math.log(2.0), device=cuda_device)
        p = math.exp(-float(lse[0]))
    else:
        lse, p = None, 1.0
    loss = top_kl_loss(row.expand(rows, V), TopLogits(values, ids, lse, 1.0 if rest else None), 1.0)
    Z = float(torch.logsumexp(row.double(), 0))
    Zr = float(torch.logsumexp(row[1:].double(), 0))
    assert abs(Z - math.log(threads)) < 1e-3
    want = p * (math.log(p) + Z) + ((1 - p) * (math.log(1 - p) - (Zr - Z)) if rest else 0.0)
    # with the rest: p Z + r (Z - Z_r), where Z and Z_r are off by the same sum
    assert abs(float(loss) - want) <= 2.0 ** -24 * ((2 + 3 + 1 + 6) * (2 if rest else 1) + abs(want))
