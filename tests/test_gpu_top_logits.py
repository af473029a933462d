"""distill.top_logits (sf_top_logits) against a stable sort and a log-sum-exp in float64.

Values and ids are equal.  The log-sum-exp: every exponential in float32 has an argument d = (x - max) / T off by 3 2^-24
|d| and rounds by 2^-23 itself; weighted by its share, |d| averages below ln V + 1 (an entropy); a thread adds at most
V / 256 + 8 of them, each sum rounding by 2^-24.  With the result's own rounding, 2^-24 of it:
  2^-24 (3 (ln V + 1) + 2 + V / 256 + 8) + 2^-24 |lse|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def check(x, k, T):
    from sparseforge_amd.distill import top_logits

    top = top_logits(x, k, T)
    V = x.shape[-1]
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    assert top.values.dtype == x.dtype and top.ids.dtype == torch.int32 and top.lse.dtype == torch.float32
    assert top.values.shape == (*x.shape[:-1], k) and top.lse.shape == x.shape[:-1] and top.temperature == T
    assert torch.equal(top.ids.long(), ids[..., :k])
    assert torch.equal(top.values.nan_to_num(nan=12345.0), values[..., :k].nan_to_num(nan=12345.0))
    lse = torch.logsumexp(x.double() / T, -1)
    plain = lse.isfinite()
    got = top.lse.double()
    assert torch.equal(got[~plain].nan_to_num(nan=12345.0), lse[~plain].nan_to_num(nan=12345.0))
    bar = 2.0 ** -24 * (3 * (math.log(V) + 1) + 2 + V / 256 + 8 + lse.abs())
    assert bool(((got - lse).abs() <= bar)[plain].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (4, 33, 7), (2, 1001, 1), (5, 1001, 1001), (3, 8192, 64),
                                      (2, 32000, 20), (3, 50257, 1024), (2, 131072, 500), (1, 262144, 1024),
                                      (700, 4099, 65), (300, 300, 300)])
def test_matches_a_stable_sort(cuda_device, dtype, rows, V, k):
    g = torch.Generator(device=cuda_device).manual_seed(V + k)
    check((torch.randn(rows, V, generator=g, device=cuda_device) * 3).to(dtype), k, 2.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_orders_that_are_hard_to_cut(cuda_device, dtype):
    """Rows of equal values, of few values, rising, falling, far apart, close together, with 0 and -0."""
    g = torch.Generator(device=cuda_device).manual_seed(7)
    V = 20011
    n = torch.arange(V, device=cuda_device).float()
    rows = [torch.full((V,), 3.25, device=cuda_device), torch.zeros(V, device=cuda_device),
            torch.where(n % 3 == 0, 0.0, -0.0), n - 9000.0, 9000.0 - n, torch.exp2(n / V * 200 - 100),
            -torch.exp2(n / V * 200 - 100), 1.0 + n * 2.0 ** -23, -1.0 - n * 2.0 ** -23,
            torch.randint(0, 4, (V,), generator=g, device=cuda_device).float(),
            torch.where(n == 12345, 5.0, -1e30), torch.randn(V, generator=g, device=cuda_device) * 1e-40,
            torch.where(n > 19000, 2.0, 1.0), torch.where(n < 1500, 2.0, 1.0)]
    x = torch.stack(rows).to(dtype)
    for k in (1, 2, 100, 700, 1024):
        check(x, k, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan(cuda_device, dtype):
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = (torch.randn(8, 3001, generator=g, device=cuda_device) * 3).to(dtype)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 77] = 2.0
    x[2, ::2] = -math.inf
    x[3, 5] = math.inf
    x[4, [9, 2000, 17]] = math.nan
    x[5] = torch.finfo(dtype).min
    x[6, 3:] = torch.finfo(dtype).min
    x[7] = math.nan
    for k in (1, 30, 1000):
        check(x, k, 2.0)


def test_views_and_shapes(cuda_device):
    from sparseforge_amd.distill import top_logits

    g = torch.Generator(device=cuda_device).manual_seed(6)
    for dtype in (torch.bfloat16, torch.float32):
        x = (torch.randn(2, 5, 3, 1003, generator=g, device=cuda_device) * 3).to(dtype)
        check(x[:, :-1, 0], 9, 2.0)           # two strides
        check(x[:, ::2, 1:, 3:1000], 9, 2.0)  # three: copied
        check(x[0, 0, 0], 4, 1.0)             # one row
        check(x.transpose(-1, -2), 2, 1.0)
        check(x[:, :1].expand(2, 4, 3, 1003), 5, 1.0)
        empty = top_logits(x[:0], 3)
        assert empty.ids.shape == (0, 5, 3, 3) and empty.lse.shape == (0, 5, 3)
    y = (torch.randn(4, 100, device=cuda_device)).requires_grad_(True)
    assert not top_logits(y, 3).values.requires_grad


def test_refusals(cuda_device):
    from sparseforge_amd.distill import top_logits

    x = torch.zeros(2, 2000, device=cuda_device)
    for k, T in ((0, 2.0), (2001, 2.0), (1025, 2.0), (5, 0.0), (5, -1.0), (5, math.nan), (5, math.inf)):
        with pytest.raises(ValueError):
            top_logits(x, k, T)
    with pytest.raises(TypeError):
        top_logits(x.half(), 3)
    with pytest.raises(RuntimeError):
        top_logits(x.cpu(), 3)
    with pytest.raises(ValueError):
        top_logits(torch.zeros(1, 262145, device=cuda_device), 3)


def test_captured_and_replayed(cuda_device):
    from sparseforge_amd.distill import top_logits

    g = torch.Generator(device=cuda_device).manual_seed(8)
    x = torch.randn(5, 32000, generator=g, device=cuda_device).bfloat16()
    top_logits(x, 64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = top_logits(x, 64)
    for _ in range(3):
        x.copy_(torch.randn(5, 32000, generator=g, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        again = top_logits(x, 64)
        assert all(torch.equal(a, b) for a, b in zip(out[:3], again[:3]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_behind_2_31_elements(cuda_device, dtype):
    """The last rows of logits whose offsets pass 32 bits."""
    from sparseforge_amd.distill import top_logits

    B, V = 8300, 262144 if dtype == torch.bfloat16 else 262143
    x = torch.zeros(B, V, dtype=dtype, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x[:, 7:1000:31] = 1.0
    x[-3:] = (torch.randn(3, V, generator=g, device=cuda_device) * 3).to(dtype)
    top = top_logits(x, 20)
    alone = top_logits(x[-3:].clone(), 20)
    assert torch.equal(top.ids[-3:], alone.ids) and torch.equal(top.values[-3:], alone.values)
    assert torch.equal(top.lse[-3:], alone.lse)
    assert bool((top.ids[:-3] == torch.arange(7, 7 + 31 * 20, 31, device=cuda_device)).all())


def test_far_apart_and_at_the_ends_of_the_temperatures(cuda_device):
    from sparseforge_amd.distill import top_logits

    x = torch.tensor([[0.0, 1.0, -2.0], [3e38, -3e38, 0.0]], device=cuda_device)
    for T in (1e-30, 1e-3, 1e30):
        top = top_logits(x, 2, T)
        assert top.ids.tolist() == [[1, 0], [0, 2]]
        want = torch.logsumexp(x.double() / T, -1).float()
        assert torch.allclose(top.lse, want, rtol=1e-6, atol=1e-6)


def test_on_two_streams(cuda_device):
    from sparseforge_amd.distill import top_logits

    g = torch.Generator(device=cuda_device).manual_seed(6)
    x = [torch.randn(300, 50257, generator=g, device=cuda_device) for _ in range(2)]
    want = [top_logits(y, 50) for y in x]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for y, stream, out in zip(x, streams, got):
            with torch.cuda.stream(stream):
                out.append(top_logits(y, 50))
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        for o in out:
            assert torch.equal(w.ids, o.ids) and torch.equal(w.values, o.values) and torch.equal(w.lse, o.lse)


def _far_apart(dev, dtype, V=30011):
    """Rows in which some logits lie far from all others, or hardly apart."""
    g = torch.Generator(device=dev).manual_seed(17)
    n = torch.randn(V, generator=g, device=dev) * 2
    i = torch.arange(V, device=dev)
    few = torch.rand(V, generator=g, device=dev) < 0.05
    rows = [torch.where(few, n, low) for low in (-1e4, -1e9, -3e38, torch.finfo(dtype).min)]
    rows += [torch.where(i % 4001 == 7, 1e4, n), torch.where(i % 97 == 7, 3e38, n), torch.where(i < 700, 100.0 + n, n),
             torch.where(i < 700, 100.0 + n, torch.where(few, n, -1e30)), n * 1e-44, torch.where(few, n * 1e-40, -1e30),
             torch.where(i == 5, 3e38, torch.where(few, n * 1e-40, -3e38)), (n * 4).round(), torch.where(few, 1.0, -1e30),
             n + torch.where(i % 2 == 0, 1e6, -1e6), torch.where(i < 1500, 2.0 + n * 1e-3, n * 1e-3 - 30.0)]
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("copies", [1, 40])  # with 1024 threads a row, with 512 and 256
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_far_from_all_others(cuda_device, dtype, copies):
    x = _far_apart(cuda_device, dtype).repeat(copies, 1)
    for k in (1, 20, 128, 300, 1000):
        check(x, k, 1.0)
