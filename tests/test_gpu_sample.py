"""logits.sample_logits (sf_sample_logits) against its definition in float64: the same token everywhere.

The kernel's exponentials are off by 2.2e-12 of themselves, and summed rounded to 2^-F of the largest, F = min(44, 60 -
ceil(log2 V)): a cumulative share is off by 2.2e-12 and V 2^-(F + 1) of the largest weight's, that where the roundings all
go one way, which they do not.  The inputs are fixed, and no draw of theirs lies within 1e-9 of a token's edge (asserted),
except where weights are equal and the sums exact.  Log-probabilities: float64 rounded once, 2^-24 of the value, and the
share's own two errors, twice.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SETTINGS = [
    {},
    {"temperature": 0.0},
    {"temperature": 0.3, "top_k": 1},
    {"temperature": 0.8, "top_k": 50, "top_p": 0.95},
    {"temperature": 1.7, "top_k": 7, "min_p": 0.3},
    {"top_p": 0.5},
    {"top_p": 0.999, "min_p": 1e-4},
    {"top_p": 0.0},
    {"temperature": 2.0, "top_k": 1500, "top_p": 0.9},
    {"min_p": 1.0},
    {"temperature": 1e-3, "top_k": 3},
    {"temperature": 30.0, "min_p": 0.05},
]


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def reference(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Token, log-probability and the draw's distance from the token's edges, of one row [V] on the CPU."""
    x = x.double()
    if bool(x.isnan().any()):
        return -1, math.nan, 1.0
    if not bool((x > -math.inf).any()):
        return -1, -math.inf, 1.0
    T, p, least = _f32(temperature), _f32(top_p), min(max(_f32(min_p), 0.0), 1.0)
    order = torch.sort(x, descending=True, stable=True).indices
    if not T > 0.0:
        order, T = order[:1], 1.0
    elif top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    w = torch.where(x[order] == top, 1.0, ((x[order] - top) / T).exp().nan_to_num(0.0)).double()
    if p < 1.0:
        before = torch.cat([w.new_zeros(1), torch.cumsum(w, 0)[:-1]])
        kept = before < p * w.sum()
        kept[0] = True
        order, w = order[kept], w[kept]
    order, w = order[w >= least], w[w >= least]
    order, at = order.sort()
    w = w[at]
    held = torch.cumsum(w, 0) / w.sum()
    u = min(max(_f32(u), 0.0), 1.0 - 2.0 ** -24)
    i = min(int((held <= u).sum()), int((w > 0).nonzero()[-1]))
    edge = min(abs(float(held[i]) - u), abs(float(held[i - 1]) - u) if i else u + 1.0)
    return int(order[i]), float((w[i] / w.sum()).log()), edge


def check(x, u, settings, edges=True):
    from sparseforge_amd.logits import sample_logits

    ids, logp = sample_logits(x, u, logprobs=True, **settings)
    B, V = x.shape
    assert ids.dtype == torch.int64 and ids.shape == (B,) and logp.dtype == torch.float32 and logp.shape == (B,)
    assert torch.equal(ids, sample_logits(x, u, **settings))
    F = min(44, 60 - math.ceil(math.log2(V)))
    for b in range(B):
        at = {n: (s[b].item() if torch.is_tensor(s) else s) for n, s in settings.items()}
        want, lp, edge = reference(x[b].cpu(), u[b].item(), **at)
        assert not edges or edge > 1e-9, "the input lies at an edge"
        assert int(ids[b]) == want, (b, at)
        got = float(logp[b])
        if math.isfinite(lp):
            assert abs(got - lp) <= 2.0 ** -24 * abs(lp) + V * 2.0 ** -F + 4.4e-12, (b, at)
        else:
            assert got == lp or (math.isnan(got) and math.isnan(lp))


def _logits(g, B, V, dtype, dev):
    x = torch.randn(B, V, generator=g, device=dev) * 3
    x[:, ::37] += torch.rand(B, x[:, ::37].shape[1], generator=g, device=dev) * 8
    return x.to(dtype)


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 33), (4, 1001), (3, 8193), (2, 32000), (3, 50257), (2, 131072)])
def test_matches_float64(cuda_device, dtype, B, V, settings):
    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = _logits(g, B, V, dtype, cuda_device)
    check(x, torch.rand(B, generator=g, device=cuda_device) * 0.999 + 0.0005, settings, edges=V > 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B", [9, 300])
def test_settings_of_each_row(cuda_device, dtype, B):
    """Tensors of settings; what lies outside a range counts as its nearest end."""
    g = torch.Generator(device=cuda_device).manual_seed(B)
    V = 5003
    x = _logits(g, B, V, dtype, cuda_device)
    temperature = torch.rand(B, generator=g, device=cuda_device) * 2
    temperature[::5] = 0.0
    top_k = torch.randint(0, 200, (B,), generator=g, device=cuda_device, dtype=torch.int32)
    top_k[1::4] = torch.tensor(-3, dtype=torch.int32)
    top_k[2::7] = V + 5
    top_p = torch.rand(B, generator=g, device=cuda_device) * 1.2
    top_p[3::8] = -0.5
    min_p = torch.rand(B, generator=g, device=cuda_device) * 0.1 - 0.02
    min_p[4::9] = 3.0
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    check(x, torch.rand(B, generator=g, device=cuda_device), settings, edges=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [6, 1000, 33000])
def test_equal_logits(cuda_device, dtype, V):
    """Ties go by the id: rows of one value, and of few values, where the sums are exact or nearly so."""
    g = torch.Generator(device=cuda_device).manual_seed(V)
    u = torch.tensor([0.0, 0.25, 0.5, 1.0 - 2.0 ** -24, 0.7], device=cuda_device)
    for settings in ({}, {"top_k": 5}, {"top_k": 5, "top_p": 0.5}, {"top_p": 0.5}, {"top_p": 0.25, "min_p": 1.0},
                     {"top_k": max(1, V // 2)}, {"temperature": 0.0}):
        check(torch.full((5, V), -2.5, device=cuda_device, dtype=dtype), u, settings, edges=False)
    few = torch.randint(-2, 2, (5, V), generator=g, device=cuda_device).to(dtype)
    few[:, 0] = 0.0
    few[:, 1] = -0.0  # equal to 0
    for settings in ({"top_k": max(1, V // 3)}, {"top_p": 0.6}, {"top_p": 0.9, "temperature": 3.0}, {"min_p": 0.2}):
        check(few, torch.rand(5, generator=g, device=cuda_device) * 0.99 + 0.003, settings, edges=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("settings", [{}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.0},
                                      {"top_k": 3000, "top_p": 0.8}])
def test_rows_with_infinities_and_nan(cuda_device, dtype, settings):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = _logits(g, 9, 3001, dtype, cuda_device)
    lowest = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 2999] = -7.0  # one token left
    x[2, torch.rand(3001, generator=g, device=cuda_device) < 0.99] = -math.inf  # fewer than top-k keeps
    x[3, 11] = math.nan
    x[4, [5, 3000]] = math.inf  # share everything
    x[5] = lowest
    x[6, 1::2] = lowest
    x[7] = math.nan
    x[8, :] = -math.inf
    x[8, 77] = math.nan
    u = torch.rand(9, generator=g, device=cuda_device)
    check(x, u, settings, edges=False)


def test_draws_follow_the_distribution(cuda_device):
    """Draws on a grid of random numbers: every token as often as its share says, within the grid's own step."""
    from sparseforge_amd.logits import sample_logits

    g = torch.Generator(device=cuda_device).manual_seed(1)
    row = torch.randn(60, generator=g, device=cuda_device) * 2
    n = 1 << 14
    u = (torch.arange(n, device=cuda_device) + 0.5) / n
    ids = sample_logits(row.expand(n, 60), u, temperature=0.7)  # a row stride of 0
    share = torch.softmax(row.double() / _f32(0.7), 0)
    assert bool((torch.bincount(ids, minlength=60) - n * share).abs().max() <= 1.0 + n * 1e-12)
    assert bool((ids[1:] >= ids[:-1]).all())


def test_strided_rows_and_odd_addresses(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32):
        wide = _logits(g, 6, 2500, dtype, cuda_device)
        u = torch.rand(3, generator=g, device=cuda_device)
        check(wide[::2, 1:2400], u, {"top_k": 20}, edges=False)   # rows from any element on
        check(wide[1::2, 3:2010], u, {"top_p": 0.8}, edges=False)
        check(wide.view(2, 3, 2500)[:, -1], u[:2], {}, edges=False)
        check(wide.t()[:3, :6], u, {}, edges=False)               # rows that are not contiguous: copied


def test_numbers_outside_the_range_count_as_its_end(cuda_device):
    from sparseforge_amd.logits import sample_logits

    x = torch.zeros(5, 4, device=cuda_device)
    u = torch.tensor([-1.0, 0.0, 1.0, 7.0, math.nan], device=cuda_device)
    assert sample_logits(x, u).tolist() == [0, 0, 3, 3, 0]


def test_refusals(cuda_device):
    from sparseforge_amd.logits import sample_logits

    x, u = torch.zeros(2, 8, device=cuda_device), torch.zeros(2, device=cuda_device)
    with pytest.raises(TypeError):
        sample_logits(x.half(), u)
    for bad in ({"temperature": -1.0}, {"temperature": math.nan}, {"top_k": -1}, {"top_p": 1.5}, {"min_p": -0.1},
                {"top_k": torch.zeros(2, device=cuda_device)}, {"top_p": torch.zeros(3, device=cuda_device)},
                {"temperature": torch.ones(2, device=cuda_device, dtype=torch.float64)}):
        with pytest.raises(ValueError):
            sample_logits(x, u, **bad)
    with pytest.raises(ValueError):
        sample_logits(x[0], u)
    with pytest.raises(ValueError):
        sample_logits(x, u.double())
    with pytest.raises(ValueError):
        sample_logits(x, u[:1])
    with pytest.raises(RuntimeError):
        sample_logits(x, u.cpu())
    with pytest.raises(RuntimeError):
        sample_logits(x, u, top_p=torch.ones(2))
    with pytest.raises(ValueError):
        sample_logits(torch.zeros(1, 262145, device=cuda_device), u[:1])
    assert sample_logits(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_longest_vocabulary(cuda_device, dtype):
    g = torch.Generator(device=cuda_device).manual_seed(9)
    x = _logits(g, 2, 262144, dtype, cuda_device)
    u = torch.tensor([0.123, 0.77], device=cuda_device)
    for settings in ({}, {"top_k": 900}, {"top_p": 0.97}, {"top_k": 200000, "top_p": 0.99}):
        check(x, u, settings)


def test_captured_and_replayed(cuda_device):
    """A captured draw replayed on new logits, numbers and settings, with eager work between: equal to eager draws."""
    from sparseforge_amd.logits import sample_logits

    g = torch.Generator(device=cuda_device).manual_seed(4)
    B, V = 3, 50257
    x, u = _logits(g, B, V, torch.bfloat16, cuda_device), torch.rand(B, generator=g, device=cuda_device)
    top_p = torch.full((B,), 0.9, device=cuda_device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sample_logits(x, u, top_p=top_p, logprobs=True)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [sample_logits(x, u, top_p=top_p, temperature=t, top_k=k, logprobs=True)
                for t, k in ((0.9, 0), (0.7, 60), (0.0, 0))]
    for i in range(4):
        x.copy_(_logits(g, B, V, torch.bfloat16, cuda_device))
        u.copy_(torch.rand(B, generator=g, device=cuda_device))
        top_p.fill_(0.5 + 0.1 * i)
        graph.replay()
        torch.cuda.synchronize()
        for (t, k), out in zip(((0.9, 0), (0.7, 60), (0.0, 0)), outs):
            again = sample_logits(x, u, top_p=top_p, temperature=t, top_k=k, logprobs=True)
            assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_whole_weight_ends_at_the_last_kept_token(cuda_device, dtype):
    """A number that counts as the last below 1 (2^-24 of the weight is more than any token's here but the largest) draws
    the last kept token of every row: sums by wave and by token agree to the unit."""
    from sparseforge_amd.logits import sample_logits

    g = torch.Generator(device=cuda_device).manual_seed(12)
    x = (torch.randn(3000, 4001, generator=g, device=cuda_device) * 2).to(dtype)
    u = torch.ones(3000, device=cuda_device)
    assert bool((sample_logits(x, u) == 4000).all())
    assert bool((sample_logits(x, u, temperature=1.3, min_p=1e-12) == 4000).all())
    # few kept: the last id among the largest n that hold the share, counted in float64
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    w = (order.values - order.values[:, :1]).exp()
    before = torch.cumsum(w, -1) - w
    kept = before < _f32(0.75) * w.sum(-1, keepdim=True)
    want = torch.where(kept, order.indices, -1).amax(-1)
    assert torch.equal(sample_logits(x, u, top_p=0.75), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extreme_temperatures_and_logits(cuda_device, dtype):
    from sparseforge_amd.logits import sample_logits

    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.tensor([[low, high, low, 0.0], [low, low, low, low], [0.0, 1.0, 1.0, -math.inf], [high, high, low, -high]],
                     device=cuda_device).to(dtype)
    u = torch.full((4,), 0.6, device=cuda_device)
    for p in (1.0, 0.9):
        for k in (0, 3):
            assert sample_logits(x, u, temperature=1e-42, top_p=p, top_k=k).tolist() == [1, 2 if k == 0 else 1, 2, 1]
    # at an infinite temperature all above -inf are alike
    assert sample_logits(x, u, temperature=math.inf).tolist() == [2, 2, 1, 2]
    assert sample_logits(x, u, temperature=math.inf, min_p=1.0).tolist() == [2, 2, 1, 2]


def test_whole_numbers_for_top_k(cuda_device):
    from sparseforge_amd.logits import sample_logits

    x, u = torch.zeros(2, 8, device=cuda_device), torch.zeros(2, device=cuda_device)
    with pytest.raises(ValueError):
        sample_logits(x, u, top_k=2.5)
    assert sample_logits(x, u, top_k=2.0).tolist() == [0, 0]


@pytest.mark.parametrize("dtype,settings", [(torch.bfloat16, {}), (torch.bfloat16, {"top_k": 40, "top_p": 0.9}),
                                            (torch.float32, {"top_p": 0.8})])
def test_rows_behind_2_31_elements(cuda_device, dtype, settings):
    """The last rows of logits whose offsets pass 32 bits, also in bytes beyond 4 GB, and of a wide stride."""
    from sparseforge_amd.logits import sample_logits

    B, V = 8300, 262144 if dtype == torch.bfloat16 else 262143
    x = torch.zeros(B, V, dtype=dtype, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x[-3:] = _logits(g, 3, V, dtype, cuda_device)
    u = torch.rand(B, generator=g, device=cuda_device)
    ids = sample_logits(x, u, **settings)
    assert torch.equal(ids[-3:], sample_logits(x[-3:].clone(), u[-3:], **settings))
    far = torch.as_strided(x, (3, 5000), (V * (B - 3) // 2, 1))
    assert torch.equal(sample_logits(far, u[:3], **settings), sample_logits(far.contiguous(), u[:3], **settings))


def test_on_another_stream_and_beside_another_draw(cuda_device):
    """Draws on two streams at once equal those in turn."""
    from sparseforge_amd.logits import sample_logits

    g = torch.Generator(device=cuda_device).manual_seed(6)
    x = [_logits(g, 40, 50257, torch.float32, cuda_device) for _ in range(2)]
    u = torch.rand(40, generator=g, device=cuda_device)
    want = [sample_logits(y, u, top_p=0.9) for y in x]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for y, stream, out in zip(x, streams, got):
            with torch.cuda.stream(stream):
                out.append(sample_logits(y, u, top_p=0.9))
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        assert all(torch.equal(w, o) for o in out)


def test_penalties_then_a_draw(cuda_device):
    """process_logits and sample_logits as a step of generation uses them: the mask's tokens only, -1 where it leaves none."""
    from sparseforge_amd.logits import process_logits, sample_logits

    g = torch.Generator(device=cuda_device).manual_seed(8)
    B, V = 6, 32000
    x = _logits(g, B, V, torch.bfloat16, cuda_device)
    history = torch.randint(0, V, (B, 50), generator=g, device=cuda_device)
    allowed = torch.rand(B, V, generator=g, device=cuda_device) < 0.01
    allowed[2] = False
    y = process_logits(x, history, repetition=1.3, allowed=allowed)
    u = torch.rand(B, generator=g, device=cuda_device)
    for settings in ({}, {"top_k": 30}, {"top_k": 500, "top_p": 0.7}, {"top_p": 0.99, "min_p": 0.01}):
        ids = sample_logits(y, u, temperature=0.9, **settings)
        assert int(ids[2]) == -1
        ok = torch.arange(B, device=cuda_device) != 2
        assert bool(allowed[ok].gather(1, ids[ok, None]).all())
        check(y, u, {"temperature": 0.9, **settings})


@pytest.mark.parametrize("settings", [{"top_k": 40}, {"top_k": 300, "top_p": 0.9}, {"top_k": 900, "temperature": 1.5},
                                      {"top_k": 2500, "top_p": 0.95}, {"top_p": 0.9}, {"top_p": 0.999}],
                         ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_far_from_all_others(cuda_device, dtype, settings):
    """Masks of -1e4, 1e9 and the type's lowest value, lone large logits, clusters, differences below 1e-30; alone and in
    rows enough for fewer threads each, which draw the same."""
    from sparseforge_amd.logits import sample_logits

    g = torch.Generator(device=cuda_device).manual_seed(17)
    V = 30011
    n = torch.randn(V, generator=g, device=cuda_device) * 2
    i = torch.arange(V, device=cuda_device)
    few = torch.rand(V, generator=g, device=cuda_device) < 0.05
    rows = [torch.where(few, n, low) for low in (-1e4, -1e9, torch.finfo(dtype).min)]
    rows += [torch.where(i % 4001 == 7, 1e4, n), torch.where(i < 700, 100.0 + n, n), n * 1e-44, (n * 4).round(),
             torch.where(few, 1.0, -1e30), torch.where(few, n - 30.0, torch.finfo(dtype).min), n * 0.5 + 12.0]
    x = torch.stack(rows).to(dtype)
    u = torch.rand(len(rows), generator=g, device=cuda_device)
    check(x, u, settings, edges=False)
    many = sample_logits(x.repeat(30, 1), u.repeat(30), **settings)
    assert torch.equal(many, sample_logits(x, u, **settings).repeat(30))
