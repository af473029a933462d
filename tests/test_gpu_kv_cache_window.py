"""A window over caches much longer than it, where the launch is cut for the whole cache: windows inside one piece of the
keys, over the edge of two, and of many.  Oracle and bar are test_gpu_kv_cache.py's."""
import pytest
import torch
from test_gpu_kv_cache import _attention, _data, _stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,group,D", [(1, 1, 64), (1, 4, 128), (8, 2, 128), (24, 1, 64), (3, 5, 200), (40, 2, 64), (150, 1, 128)])
def test_window_in_a_long_cache(cuda_device, n, group, D):
    from sparseforge_amd import _lib as L
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n + D)
    B, Hk, held = 2, 2, [30000, 1700]
    T = max(held) + n
    k, v = _data(g, B, T, Hk, D, cuda_device)
    q = torch.randn(B, n, group * Hk, D, generator=g, device=cuda_device).bfloat16()
    cache = KVCache8(B, Hk, D, T)
    cache.extend(max(held), torch.tensor(held, dtype=torch.int32, device=cuda_device))
    cache.append(k[:, :max(held)], v[:, :max(held)])
    cache.extend(n)
    cache.append(*(torch.stack([x[b, h:h + n] for b, h in enumerate(held)]) for x in (k, v)))
    assert L.lib().sf_kv8_attend_workspace_size(B, Hk, group * Hk, D, n, cache.bound) > 0  # keys in several pieces
    kept = [[_stored(x[b], h + n) for x in (k, v)] for b, h in enumerate(held)]
    for window in (1, 64, 200, 1000, 5000, 20000, 29000):
        out = cache.attend(q, window=window).view(B, n, group * Hk, D).double()
        for b, h in enumerate(held):
            o, bar = _attention(q[b], *kept[b], h, D ** -0.5, window)
            assert bool(((out[b] - o).abs() <= bar).all()), (window, b)
