"""Attention over the 8-bit cache at the ends of the numbers' range: values as large as bf16 holds, value scales of
neighbouring blocks far apart.  Oracle and bar are test_gpu_kv_cache.py's."""
import pytest
import torch
from test_gpu_kv_cache import BLOCK, _attention, _data, _stored

pytestmark = pytest.mark.gpu


def _outputs(q, k, v, D):
    """Attention of the last q.shape[1] tokens of k, v over all of them: (out, o, bar) [n, H, D]."""
    from sparseforge_amd.kv_cache import KVCache8

    n, H, T = q.shape[1], q.shape[2], k.shape[1]
    cache = KVCache8(1, k.shape[2], D, T)
    if T > n:
        cache.extend(T - n)
        cache.append(k[:, :T - n], v[:, :T - n])
    cache.extend(n)
    cache.append(k[:, T - n:], v[:, T - n:])
    out = cache.attend(q).view(n, H, D).double()
    return out, *_attention(q[0], _stored(k[0], T), _stored(v[0], T), T - n, D ** -0.5, 0)


# few rows and many, one piece of the keys and several, ending on a block's edge and inside a block
FORMS = [(1, 1, 64, 6 * BLOCK), (1, 4, 128, 6 * BLOCK + 20), (1, 1, 128, 5000), (24, 1, 128, 700), (40, 4, 64, 500),
         (40, 4, 128, 6 * BLOCK), (150, 1, 128, 5000), (9, 2, 200, 2100), (200, 2, 256, 1000)]


@pytest.mark.parametrize("n,group,D,T", FORMS)
def test_largest_values(cuda_device, n, group, D, T):
    """Values between half of and the largest that bf16 has: a sum of few of them passes the floats, their mean does not."""
    g = torch.Generator(device=cuda_device).manual_seed(n + T)
    Hk = 2
    k, v = _data(g, 1, T, Hk, D, cuda_device)
    v = ((1.0 + 0.98 * torch.rand(v.shape, generator=g, device=cuda_device)) * 2.0 ** 127).bfloat16()
    v[:, :, 1] *= -1.0
    q = torch.randn(1, n, group * Hk, D, generator=g, device=cuda_device).bfloat16()
    for size in (1.0, 0.0):  # and all weights equal
        out, o, bar = _outputs(q * size, k, v, D)
        assert bool(((out - o).abs() <= bar).all()), float(((out - o).abs() / bar).max())


@pytest.mark.parametrize("n,group,D,T", FORMS)
def test_large_values_without_weight(cuda_device, n, group, D, T):
    """A block in the middle whose values are 2^80 times the others' and whose keys score too low to have any weight."""
    g = torch.Generator(device=cuda_device).manual_seed(n * T)
    Hk = 2
    k, v = _data(g, 1, T, Hk, D, cuda_device)
    q = torch.randn(1, n, group * Hk, D, generator=g, device=cuda_device).bfloat16()
    q[..., 0] = 64.0
    k[..., 0] = 1.0
    k[:, 2 * BLOCK:3 * BLOCK, :, 0] = -64.0
    v[:, 2 * BLOCK:3 * BLOCK] = (v[:, 2 * BLOCK:3 * BLOCK].float() * 2.0 ** 80).bfloat16()
    out, o, bar = _outputs(q, k, v, D)
    assert float(o.abs().max()) < 100.0
    assert bool(((out - o).abs() <= bar).all()), float(((out - o).abs() / bar).max())


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("down", [12, 24, 36, 60])
def test_small_weights_beside_a_large_one(cuda_device, n, down):
    """One key with values of 0 and nearly all of the weight, 60000 with 2^-down of it each: the output is what these add,
    and the bar, which is in terms of what adds, holds for it."""
    g = torch.Generator(device=cuda_device).manual_seed(down)
    T, D = 60000, 64
    k = torch.zeros(1, T, 1, D, dtype=torch.bfloat16, device=cuda_device)
    k[0, 3, 0, 0] = 1.0
    v = (1.0 + torch.rand(1, T, 1, D, generator=g, device=cuda_device)).bfloat16()
    v[0, 3] = 0.0
    q = torch.zeros(1, n, 2, D, dtype=torch.bfloat16, device=cuda_device)
    q[..., 0] = 0.6931472 * down * D ** 0.5
    out, o, bar = _outputs(q, k, v, D)
    assert bool(((out - o).abs() <= bar).all()), float(((out - o).abs() / bar).max())


@pytest.mark.parametrize("n,group,D,T", FORMS)
def test_scores_of_next_to_nothing(cuda_device, n, group, D, T):
    """Keys and a scale whose product no float holds: every score is 0 within 2^-100, hidden keys stay hidden."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n + D)
    k, v = _data(g, 1, T, 2, D, cuda_device)
    k = (k.float() * 1e-38 * 1e-2).bfloat16()
    assert 0 < float(k.abs().max()) < 1e-38
    q = torch.randn(1, n, group * 2, D, generator=g, device=cuda_device).bfloat16()
    cache = KVCache8(1, 2, D, T + n)
    if T > n:
        cache.extend(T - n)
        cache.append(k[:, :T - n], v[:, :T - n])
    cache.extend(n)
    cache.append(k[:, T - n:], v[:, T - n:])
    for window in (0, 100):
        out = cache.attend(q, scale=1e-12, window=window).view(n, 2 * group, D).double()
        o, bar = _attention(q[0] * 0, _stored(k[0], T), _stored(v[0], T), T - n, 1.0, window)
        assert bool(((out - o).abs() <= bar).all())


@pytest.mark.parametrize("n,group,D,T", FORMS)
def test_scales_past_the_floats(cuda_device, n, group, D, T):
    """A scale, or a scale times a key's, above every float: rows that score 0 everywhere weigh all keys alike."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n - D)
    k, v = _data(g, 1, T, 2, D, cuda_device)
    q = torch.zeros(1, n, group * 2, D, dtype=torch.bfloat16, device=cuda_device)
    for size, scale in ((1.0, 3e38), (1e-3, 2.9e38), (1e30, 1e30)):
        cache = KVCache8(1, 2, D, T + n)
        x = (k.float() * size).bfloat16()
        if T > n:
            cache.extend(T - n)
            cache.append(x[:, :T - n], v[:, :T - n])
        cache.extend(n)
        cache.append(x[:, T - n:], v[:, T - n:])
        out = cache.attend(q, scale=scale).view(n, 2 * group, D).double()
        o, bar = _attention(q[0], _stored(k[0], T), _stored(v[0], T), T - n, 1.0, 0)
        assert bool(((out - o).abs() <= bar).all())


@pytest.mark.parametrize("n,group,D,T", [(1, 1, 64, 33), (1, 4, 128, 63), (20, 4, 64, 40), (50, 1, 128, 50), (7, 2, 200, 30)])
def test_an_incomplete_block_alone(cuda_device, n, group, D, T):
    """Fewer than 64 tokens are held as they came and weighed with 16 bits: errors of 2^-17 of a weight, spread evenly, are
    1 % of what storing the output in bf16 makes in the root of the mean square, which some 500 outputs and more, whose
    roundings are independent of them, show to a few in a thousand."""
    g = torch.Generator(device=cuda_device).manual_seed(3 * n + T)
    k, v = _data(g, 1, T, 8, D, cuda_device)
    q = torch.randn(1, n, group * 8, D, generator=g, device=cuda_device).bfloat16()
    out, o, _ = _outputs(q, k, v, D)
    least = (o.bfloat16().double() - o).pow(2).mean().sqrt()
    assert float((out - o).pow(2).mean().sqrt() / least) < 1.01


@pytest.mark.parametrize("n,group,D,window", [(200, 1, 128, 0), (90, 2, 64, 0), (24, 4, 128, 0), (60, 2, 200, 0),
                                              (200, 1, 64, 100), (8, 2, 128, 40)])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -60])
def test_largest_values_out_of_sight(cuda_device, n, group, D, window, size):
    """The largest numbers of bf16 in tokens that some rows see and others of the same wave do not: theirs are as they are
    without them."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n + D)
    T, Hk = 260 + n, 2
    k, v = _data(g, 1, T, Hk, D, cuda_device)
    v = (v.float() * size).bfloat16()
    # the last block of codes but one, or the first that a window leaves
    at = 192 if window else (T // BLOCK - 1) * BLOCK
    v[:, at:at + BLOCK] = 3.3e38 * torch.sign(v[:, at:at + BLOCK])
    q = torch.randn(1, n, group * Hk, D, generator=g, device=cuda_device).bfloat16()
    cache = KVCache8(1, Hk, D, T)
    cache.extend(T - n)
    cache.append(k[:, :T - n], v[:, :T - n])
    cache.extend(n)
    cache.append(k[:, T - n:], v[:, T - n:])
    out = cache.attend(q, window=window).view(n, group * Hk, D).double()
    o, bar = _attention(q[0], _stored(k[0], T), _stored(v[0], T), T - n, D ** -0.5, window)
    assert bool(((out - o).abs() <= bar).all()), float(((out - o).abs() / bar).max())
