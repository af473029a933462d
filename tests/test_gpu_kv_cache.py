"""kv_cache.KVCache8 (sf_kv8_append, sf_kv8_values, sf_kv8_attend) against its definition in float64.

values: a whole block's values are code * scale with the codes of exact arithmetic and scale = max|x| / 127 rounded to
float32, the product rounded once more: 2^-23 of the value at most.  Rows of an incomplete block are equal.

attend, with w_j the softmax's weights and A = sum_j w_j |v_j| over the values the cache stands for: the weights round to
bf16 as operands (2^-8 A at most), the output is rounded once (2^-8 |o|); in float32 a score is off by at most
(D + 4) 2^-24 scale sum_d |q_d k_jd| =: d and so a weight by 2 d of itself against the others; exp2, the sums and the
scales stay below 2^-18 A together for the lengths here.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = 64


def _stored(x, end):
    """The first `end` rows of x [T, H, D] as the cache holds them, float64."""
    y = x[:end].double().clone()
    for at in range(0, end // BLOCK * BLOCK, BLOCK):
        z = y[at:at + BLOCK]
        top = z.abs().amax((0, 2), keepdim=True)
        y[at:at + BLOCK] = torch.where(top > 0, torch.round(127 * z / top) * top / 127, z)
    return y


def _attention(q, k, v, start, scale, window):
    """q [n, H, D] at positions start.., k and v [T, Hk, D] float64 -> (o, bar) [n, H, D]."""
    n, H, D = q.shape
    group = H // k.shape[1]
    q = q.double()
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("nhd,thd->hnt", q, k) * scale
    size = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()) * scale
    at = start + torch.arange(n, device=q.device)[:, None]
    key = torch.arange(k.shape[0], device=q.device)[None]
    hidden = key > at
    if window:
        hidden |= key <= at - window
    w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    o = torch.einsum("hnt,thd->nhd", w, v)
    A = torch.einsum("hnt,thd->nhd", w, v.abs())
    d = ((D + 4) * 2.0 ** -24 * size.masked_fill(hidden, 0.0).amax(-1)).T[..., None]
    return o, (2.0 ** -8 + 4 * d + 2.0 ** -18) * A + 2.0 ** -8 * o.abs()


def _data(g, B, T, Hk, D, dev):
    k = torch.randn(B, T, Hk, D, generator=g, device=dev) * (1 + 3 * (torch.rand(Hk, D, generator=g, device=dev) < 0.1))
    return k.bfloat16(), torch.randn(B, T, Hk, D, generator=g, device=dev).bfloat16()


def _fill(cache, k, v, lengths):
    """k, v [B, T, ..] into an empty cache, lengths[b] of them."""
    dev = k.device
    if k.shape[1]:
        cache.extend(k.shape[1], torch.tensor(lengths, dtype=torch.int32, device=dev))
        for layer in range(cache.layers):
            cache.append(k, v, layer)


@pytest.mark.parametrize("D", [8, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("lengths", [(1,), (63, 64, 65), (0, 128, 200), (130, 1, 64)])
def test_values(cuda_device, D, lengths):
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(D + sum(lengths))
    B, T, Hk = len(lengths), max(lengths), 3
    k, v = _data(g, B, T, Hk, D, cuda_device)
    cache = KVCache8(B, Hk, D, T + 70)
    _fill(cache, k, v, lengths)
    got = cache.values(tokens=T + 3)
    for b, end in enumerate(lengths):
        for y, x in zip(got, (k, v)):
            want = _stored(x[b], end)
            full = end // BLOCK * BLOCK
            assert bool(((y[b, :full].double() - want[:full]).abs() <= want[:full].abs() * 2.0 ** -23).all())
            assert torch.equal(y[b, full:end].double(), want[full:])
            assert not y[b, end:].any()
    # another first position for each sequence
    first = torch.tensor([max(0, n - 5) for n in lengths], dtype=torch.int32, device=cuda_device)
    part = cache.values(first, 7)
    for b, f in enumerate(first.tolist()):
        for y, p in zip(got, part):
            n = min(7, y.shape[1] - f)
            assert torch.equal(p[b, :n], y[b, f:f + n]) and not p[b, n:].any()


def test_rows_one_at_a_time_and_together_give_the_same_cache(cuda_device):
    """200 tokens in one step, one a step, and in odd pieces; strided rows, two layers, ragged counts."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(3)
    B, T, Hk, D = 3, 200, 2, 80
    rows = torch.randn(B, T, 2 * Hk * D, generator=g, device=cuda_device).bfloat16()
    k, v = rows[..., :Hk * D].view(B, T, Hk, D), rows[..., Hk * D:].view(B, T, Hk, D)
    want = None
    for pieces in ([200], [1] * 200, [3, 61, 1, 70, 65], [130, 70], [64, 64, 64, 8], [63, 129, 8]):
        cache = KVCache8(B, Hk, D, T, layers=2)
        at = 0
        for n in pieces:
            cache.extend(n)
            for layer in (0, 1):
                cache.append(k[:, at:at + n], (v if layer == 0 else k)[:, at:at + n], layer)
            at += n
        got = (*cache.values(), *cache.values(layer=1))
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert cache.ends.tolist() == [T] * B and cache.bound == T
    # each sequence at its own pace: b takes b + 1 tokens a step
    cache = KVCache8(B, Hk, D, T * 3)
    done = [0] * B
    for _ in range(66):
        counts = torch.tensor([b + 1 for b in range(B)], dtype=torch.int32, device=cuda_device)
        piece = [torch.stack([torch.cat([x[b], x[b, :3]])[d:d + 3] for b, d in enumerate(done)]) for x in (k, v)]
        cache.extend(3, counts)
        cache.append(*piece)
        done = [d + b + 1 for b, d in enumerate(done)]
    got = cache.values(tokens=T)
    for b in range(B):
        whole = done[b] // BLOCK * BLOCK
        assert torch.equal(got[0][b, :whole], want[0][b, :whole]) and torch.equal(got[1][b, :whole], want[1][b, :whole])


@pytest.mark.parametrize("top", [2.0 ** -126, 2.0 ** -130, 3e-30, 1.0, 2.0 ** 64, 3.38e38])
def test_values_of_extreme_size(cuda_device, top):
    """The smallest and the largest numbers, ties of the rounding (half the largest), zero blocks."""
    from sparseforge_amd.kv_cache import KVCache8

    D = 64
    x = torch.zeros(1, 2 * BLOCK, 1, D, device=cuda_device)
    x[0, :BLOCK, 0] = torch.linspace(-1, 1, BLOCK * D, device=cuda_device).view(BLOCK, D) * top
    x[0, 0, 0, :3] = torch.tensor([top, top / 2, -top / 2], device=cuda_device)
    x = x.bfloat16()
    cache = KVCache8(1, 1, D, 2 * BLOCK)
    _fill(cache, x, x, [2 * BLOCK])
    want = _stored(x[0], 2 * BLOCK)
    tiny = 127 * 2.0 ** -149  # a scale below the normal numbers is a multiple of 2^-149
    for y in cache.values():
        assert bool(((y[0].double() - want).abs() <= want.abs() * 2.0 ** -23 + (tiny if top < 1e-36 else 0)).all())
        assert not y[0, BLOCK:].any()


CASES = [
    # B, n, H, Hk, D, held, window
    (1, 1, 4, 4, 64, (0,), 0),
    (1, 1, 32, 32, 64, (32,), 0),
    (3, 1, 8, 2, 128, (63, 64, 700), 0),
    (2, 1, 6, 1, 80, (1000, 5), 0),
    (1, 1, 16, 1, 128, (5000,), 0),
    (1, 1, 40, 1, 64, (333,), 0),
    (2, 5, 8, 8, 64, (300, 61), 0),
    (2, 7, 12, 4, 128, (130, 1), 0),
    (1, 3, 24, 2, 256, (100,), 0),
    (1, 17, 3, 3, 200, (64,), 0),
    (1, 129, 8, 2, 128, (0,), 0),
    (2, 200, 4, 2, 64, (77, 300), 0),
    (1, 65, 3, 1, 40, (63,), 0),
    (2, 1, 4, 2, 64, (300, 20), 64),
    (2, 1, 4, 2, 128, (300, 20), 1),
    (1, 90, 4, 1, 64, (200,), 33),
    (1, 90, 4, 4, 128, (200,), 100),
    (1, 300, 5, 1, 128, (1500,), 700),
]


# every form of heads and rows: one row a head, 16, 17, 32, 33, 128, 129 and many, with keys in one piece and in several
CASES += [(2, n, 2, 1, D, held, 0) for D in (64, 128, 136, 192, 248) for n, held in
          ((1, (200, 3000)), (8, (2000, 5)), (9, (700, 64)), (16, (1300, 63)), (17, (2500, 1)), (64, (0, 900)),
           (65, (400, 4000)), (150, (1, 1100)))]
CASES += [(1, 100, 6, 2, D, (900,), 150) for D in (136, 256)]


@pytest.mark.parametrize("B,n,H,Hk,D,held,window", CASES)
def test_attend(cuda_device, B, n, H, Hk, D, held, window):
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n * 1000 + D + sum(held))
    T = max(held) + n
    k, v = _data(g, B, T, Hk, D, cuda_device)
    q = torch.randn(B, n, H, D, generator=g, device=cuda_device).bfloat16()
    # the last sequence of a batch brings fewer tokens, one that has ended none
    counts = [n] * B
    if B > 1:
        counts[-1] = n // 2
    cache = KVCache8(B, Hk, D, T + 1)
    _fill(cache, k[:, :max(held)], v[:, :max(held)], held)
    cache.extend(n, torch.tensor(counts, dtype=torch.int32, device=cuda_device))
    cache.append(torch.stack([k[b, h:h + n] for b, h in enumerate(held)]),
                 torch.stack([v[b, h:h + n] for b, h in enumerate(held)]))
    for scale in (None, 0.3):
        out = cache.attend(q, scale=scale, window=window).view(B, n, H, D).double()
        for b in range(B):
            c, end = counts[b], held[b] + counts[b]
            assert not out[b, c:].any()
            if c:
                o, bar = _attention(q[b, :c], _stored(k[b], end), _stored(v[b], end), held[b], scale or D ** -0.5, window)
                assert bool(((out[b, :c] - o).abs() <= bar).all()), float(((out[b, :c] - o).abs() / bar).max())


def test_attend_strided_queries_and_odd_addresses(cuda_device):
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(5)
    B, n, H, Hk, D = 2, 4, 6, 2, 64
    k, v = _data(g, B, 70, Hk, D, cuda_device)
    cache = KVCache8(B, Hk, D, 100)
    _fill(cache, k, v, [70, 70])
    cache.extend(n)
    fused = torch.randn(B, n, (H + 2 * Hk) * D + 3, generator=g, device=cuda_device).bfloat16()
    for off in (0, 3):  # an offset of 3 elements is copied to an aligned place
        f = fused[..., off:off + (H + 2 * Hk) * D]
        q = f[..., :H * D].unflatten(-1, (H, D))
        cache.append(f[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)), f[..., (H + Hk) * D:].unflatten(-1, (Hk, D)))
        a = cache.attend(q)
        cache.append(f[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)).contiguous(),
                     f[..., (H + Hk) * D:].unflatten(-1, (Hk, D)).contiguous())
        assert torch.equal(a, cache.attend(q.contiguous()))
        assert torch.equal(a, cache.attend(q.transpose(1, 2).contiguous().transpose(1, 2)))


@pytest.mark.parametrize("n,held", [(1, 100), (100, 30), (40, 90)])
def test_nothing_past_the_end_or_out_of_sight_reaches_an_output(cuda_device, n, held):
    """Storage full of NaN before the first row; NaN and infinities in one token: exactly the queries that see it, or a
    key of the block that it has completed, are NaN."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n)
    Hk, H, D, T = 2, 4, 64, held + n
    k, v = _data(g, 1, T, Hk, D, cuda_device)
    q = torch.randn(1, n, H, D, generator=g, device=cuda_device).bfloat16()

    def outputs(k, v, window=0):
        cache = KVCache8(1, Hk, D, 400)
        for t in (cache.k_scales, cache.v_scales, cache.k_tail, cache.v_tail):
            t.fill_(math.nan)
        cache.k_codes.fill_(127)
        cache.v_codes.fill_(-127)
        cache.extend(held)
        cache.append(k[:, :held], v[:, :held])
        cache.extend(n)
        cache.append(k[:, held:], v[:, held:])
        return cache.attend(q, window=window).view(n, H, D)

    clean = outputs(k, v)
    assert not clean.isnan().any()
    whole = T // BLOCK * BLOCK
    for where in (T - 1, T - 3, held, 5, 64):
        for value in (math.nan, math.inf, -math.inf):
            for window in (0, 20):
                base = clean if not window else outputs(k, v, window)
                for x in (k, v):
                    x2 = x.clone()
                    x2[0, where, 1, 7] = value  # of key-value head 1: query heads 2 and 3
                    got = outputs(x2 if x is k else k, x2 if x is v else v, window)
                    assert torch.equal(got[:, :2], base[:, :2])
                    b0 = where // BLOCK * BLOCK
                    lo, hi = (b0, b0 + BLOCK) if where < whole else (where, where + 1)  # keys that are NaN
                    at = held + torch.arange(n, device=cuda_device)
                    sees = at >= lo
                    if window:
                        sees &= at - window < hi - 1
                    assert bool(got[sees][:, 2:].isnan().all())
                    assert torch.equal(got[~sees], base[~sees])


def test_runaway_and_flat_scores(cuda_device):
    """Scores of thousands, where one key takes all, and of exactly 0, where all are equal; a maximum that rises over
    blocks in small and in large steps."""
    from sparseforge_amd.kv_cache import KVCache8

    D, T = 64, 500
    g = torch.Generator(device=cuda_device).manual_seed(1)
    v = torch.randn(1, T, 1, D, generator=g, device=cuda_device).bfloat16()
    ramp = torch.linspace(0, 1, T, device=cuda_device)[None, :, None, None]
    one = torch.ones(1, T, 1, D, device=cuda_device)
    for k, size in ((one * ramp, 1.0), (one * ramp, 40.0), (one * ramp, -40.0), (one * ramp, 3e4), (one * 0, 5.0),
                    (one * ramp.flip(1), 3e4), (one * (ramp * 300).floor() / 300, 2.0)):
        k = k.bfloat16()
        q = (torch.ones(1, 1, 1, D, device=cuda_device) * size).bfloat16()
        cache = KVCache8(1, 1, D, T)
        _fill(cache, k, v, [T - 1])
        cache.extend(1)
        cache.append(k[:, -1:], v[:, -1:])
        out = cache.attend(q).view(1, 1, D).double()
        o, bar = _attention(q[0], _stored(k[0], T), _stored(v[0], T), T - 1, D ** -0.5, 0)
        assert bool(((out - o).abs() <= bar).all())


@pytest.mark.parametrize("n", [1, 40])
def test_values_of_any_size(cuda_device, n):
    """Blocks of values from 2^-100 to 2^110, of zeros, and all in one sequence: the smallest ones carry the weight of
    their keys, and a block of large ones that has next to none of it adds next to nothing."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(n)
    T, H, Hk, D = 6 * BLOCK + 20, 4, 2, 64
    k, v = _data(g, 1, T, Hk, D, cuda_device)
    q = torch.randn(1, n, H, D, generator=g, device=cuda_device).bfloat16()
    mixed = torch.tensor([2.0 ** e for e in (0, -100, 90, -66, 66, 0, 0)], device=cuda_device)
    mixed[5] = 0.0
    for size in (torch.full((7,), 2.0 ** -100, device=cuda_device), torch.full((7,), 2.0 ** 110, device=cuda_device),
                 torch.zeros(7, device=cuda_device), mixed, mixed.flip(0)):
        w = (v.float() * size.repeat_interleave(BLOCK)[:T, None, None]).bfloat16()
        cache = KVCache8(1, Hk, D, T)
        if T > n:
            _fill(cache, k[:, :T - n], w[:, :T - n], [T - n])
        cache.extend(n)
        cache.append(k[:, T - n:], w[:, T - n:])
        out = cache.attend(q).view(n, H, D).double()
        o, bar = _attention(q[0], _stored(k[0], T), _stored(w[0], T), T - n, D ** -0.5, 0)
        assert bool(((out - o).abs() <= bar).all())


def test_captured_step_replayed(cuda_device):
    """One token's step as a graph, replayed from 60 tokens to 70 (a block is completed on the way) with eager work and
    waits between the replays, each against the same step without a graph."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(12)
    B, H, Hk, D, T = 2, 4, 2, 64, 72
    k, v = _data(g, B, T, Hk, D, cuda_device)
    q = torch.randn(T, B, 1, H, D, generator=g, device=cuda_device).bfloat16()
    plain, caught = KVCache8(B, Hk, D, T), KVCache8(B, Hk, D, T)
    for c in (plain, caught):
        _fill(c, k[:, :60], v[:, :60], [60, 60])
    now = [torch.empty_like(x) for x in (q[0], k[:, :1], v[:, :1])]

    def step(c):
        c.extend(1)
        c.append(now[1], now[2])
        return c.attend(now[0])

    step(KVCache8(B, Hk, D, T))  # the kernels are loaded before the capture
    torch.cuda.synchronize()
    caught.bound = T - 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caught)
    for i in range(60, 70):
        for x, y in zip(now, (q[i], k[:, i:i + 1], v[:, i:i + 1])):
            x.copy_(y)
        plain.bound = T - 1  # the same cut of the launch
        want = step(plain)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        torch.randn(1000, device=cuda_device).sum().item()
    assert caught.ends.tolist() == [70, 70]
    assert all(torch.equal(a, b) for a, b in zip(caught.values(0, 70), plain.values(0, 70)))


def test_queries_that_are_not_finite_stay_with_their_rows(cuda_device):
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(2)
    k, v = _data(g, 1, 300, 2, 64, cuda_device)
    q = torch.randn(1, 1, 8, 64, generator=g, device=cuda_device).bfloat16()
    cache = KVCache8(1, 2, 64, 300)
    _fill(cache, k[:, :299], v[:, :299], [299])
    cache.extend(1)
    cache.append(k[:, 299:], v[:, 299:])
    clean = cache.attend(q).view(8, 64)
    for value in (math.nan, math.inf):
        q2 = q.clone()
        q2[0, 0, 5, 3] = value
        got = cache.attend(q2).view(8, 64)
        assert bool(got[5].isnan().all())
        keep = [i for i in range(8) if i != 5]
        assert torch.equal(got[keep], clean[keep])


def test_offsets_past_32_bits(cuda_device):
    """The second sequence's codes begin more than 2^31 bytes into theirs."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(6)
    B, Hk, D, T = 2, 1, 256, 150
    cache = KVCache8(B, Hk, D, (2 ** 31 // 256) + 1000)
    small = KVCache8(B, Hk, D, T)
    k, v = _data(g, B, T, Hk, D, cuda_device)
    q = torch.randn(B, 1, 4, D, generator=g, device=cuda_device).bfloat16()
    for c in (cache, small):
        _fill(c, k[:, :T - 1], v[:, :T - 1], [T - 1, T - 1])
        c.extend(1)
        c.append(k[:, T - 1:], v[:, T - 1:])
    assert all(torch.equal(a, b) for a, b in zip(cache.values(), small.values()))
    assert torch.equal(cache.attend(q), small.attend(q))


def test_more_keys_than_the_bound_are_read(cuda_device):
    """The launch is sized by `bound`; counters that have moved on without the host (a replayed graph) are read."""
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(9)
    k, v = _data(g, 2, 3000, 2, 64, cuda_device)
    q = torch.randn(2, 1, 4, 64, generator=g, device=cuda_device).bfloat16()
    cache = KVCache8(2, 2, 64, 3000)
    _fill(cache, k[:, :2999], v[:, :2999], [2999, 1500])
    cache.extend(1)
    cache.append(k[:, 2999:], v[:, 2999:])
    want = cache.attend(q).double()
    for bound in (1, 700, 1500):
        cache.bound = bound
        got = cache.attend(q).double()
        assert bool(((got - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -8 * want.abs().max()).all())


def test_on_another_stream(cuda_device):
    from sparseforge_amd.kv_cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(11)
    k, v = _data(g, 1, 300, 2, 128, cuda_device)
    q = torch.randn(1, 1, 8, 128, generator=g, device=cuda_device).bfloat16()

    def whole():
        cache = KVCache8(1, 2, 128, 300)
        _fill(cache, k[:, :299], v[:, :299], [299])
        cache.extend(1)
        cache.append(k[:, 299:], v[:, 299:])
        return cache.attend(q)

    want = whole()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = whole()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals(cuda_device):
    from sparseforge_amd.kv_cache import KVCache8

    dev = cuda_device
    for bad in ((0, 1, 64, 10), (1, 0, 64, 10), (1, 1, 64, 0), (1, 1, 60, 10), (1, 1, 264, 10), (1, 1, 0, 10)):
        with pytest.raises(ValueError):
            KVCache8(*bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        KVCache8(1, 1, 64, 10, device="cpu")
    cache = KVCache8(2, 2, 64, 100)  # 128 with whole blocks
    k = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        cache.append(k, k)  # no step under way
    with pytest.raises(ValueError):
        cache.extend(129)
    with pytest.raises(ValueError):
        cache.extend(0)
    with pytest.raises(ValueError):
        cache.extend(4, torch.zeros(3, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        cache.extend(4, torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError):
        cache.extend(4, torch.zeros(2, dtype=torch.int32))
    assert cache.bound == 0
    cache.extend(4)
    cache.append(k, k)
    for bad in (k[:, :3], k[:1], k[..., :32], torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16, device=dev), k[0]):
        with pytest.raises(ValueError):
            cache.append(bad, k)
        with pytest.raises(ValueError):
            cache.append(k, bad)
    with pytest.raises(TypeError):
        cache.append(k.float(), k)
    with pytest.raises(RuntimeError):
        cache.append(k.cpu(), k)
    with pytest.raises(TypeError):
        cache.attend(k.float())
    with pytest.raises(ValueError):
        cache.attend(torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16, device=dev))  # 3 heads over 2
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            cache.attend(k, scale=scale)
    with pytest.raises(ValueError):
        cache.attend(k, window=-1)
    with pytest.raises(IndexError):
        cache.attend(k, layer=1)
    with pytest.raises(ValueError):
        cache.values(tokens=129)
    with pytest.raises(ValueError):
        cache.values(torch.zeros(3, dtype=torch.int32, device=dev), 4)
    cache.reset()
    assert cache.ends.tolist() == [0, 0] and cache.bound == 0
