"""logits.process_logits (sf_process_logits) against its definition in float64.

Bar, per element: each of at most five float32 operations (quotient or product, frequency times count, two
differences, the bias) rounds by 2^-24 of what it gives, each at most the sum of the magnitudes S that enter:
5 * 2^-24 S; storing in bf16 moves the result by 2^-8 of itself more.  Untouched logits and -inf are equal.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _bits(mask):
    """bool [.., V] -> int32 [.., ceil(V / 32)]"""
    V = mask.shape[-1]
    pad = torch.zeros(*mask.shape[:-1], -(-V // 32) * 32, dtype=torch.int64, device=mask.device)
    pad[..., :V] = mask
    words = (pad.unflatten(-1, (-1, 32)) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def _reference(x, history, lengths, rep, pres, freq, bias, allowed):
    y, S = x.double().clone(), x.double().abs()
    B, V = x.shape
    for b in range(B):
        ids = history[b].long()
        if lengths is not None:
            ids = ids[:max(0, int(lengths[b]))]
        ids = ids[(ids >= 0) & (ids < V)]
        c = torch.bincount(ids, minlength=V).double()
        met = c > 0
        r, p, f = (float(t[b]) if torch.is_tensor(t) else t for t in (rep, pres, freq))
        r = float(torch.tensor(r, dtype=torch.float32))
        p, f = float(torch.tensor(p, dtype=torch.float32)), float(torch.tensor(f, dtype=torch.float32))
        z = torch.where(y[b] > 0, y[b] / r, y[b] * r)
        S[b] = torch.where(met, S[b] + z.abs() + f * c + abs(p), S[b])
        y[b] = torch.where(met, z - f * c - p, y[b])
    if bias is not None:
        S = S + bias.double().abs()
        y = y + bias.double()
    if allowed is not None:
        y = y.masked_fill(~allowed, -math.inf)
    return y, S


def _close(got, y, S):
    finite = y.isfinite()
    assert torch.equal(got.double()[~finite], y[~finite])
    bar = 5 * 2.0 ** -24 * S + (2.0 ** -8 * y.abs() if got.dtype == torch.bfloat16 else 0.0)
    assert bool(((got.double() - y).abs() <= bar)[finite].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V,n", [(1, 1, 1), (1, 7, 3), (2, 33, 500), (3, 2048, 1), (2, 32000, 700), (5, 50257, 1500),
                                   (40, 1001, 90), (300, 257, 20), (1, 131072, 9000)])
def test_matches_float64(cuda_device, dtype, B, V, n):
    from sparseforge_amd.logits import process_logits

    g = torch.Generator(device=cuda_device).manual_seed(V + n)
    x = (torch.randn(B, V, generator=g, device=cuda_device) * 3).to(dtype)
    history = torch.randint(0, max(1, V // 2), (B, n), generator=g, device=cuda_device)
    history[:, ::7] = -1
    history[:, 3::11] = V
    history[0, 1::5] = 2 ** 40  # ids far outside
    lengths = torch.randint(-1, n + 4, (B,), generator=g, device=cuda_device, dtype=torch.int32)
    rep = 1 + torch.rand(B, generator=g, device=cuda_device)
    pres = torch.rand(B, generator=g, device=cuda_device)
    freq = torch.rand(B, generator=g, device=cuda_device)
    bias = torch.randn(B, V, generator=g, device=cuda_device)
    allowed = torch.rand(B, V, generator=g, device=cuda_device) < 0.6
    allowed[0] = False  # nothing may follow
    _close(process_logits(x, history, lengths, repetition=rep, presence=pres, frequency=freq, bias=bias,
                          allowed=allowed), *_reference(x, history, lengths, rep, pres, freq, bias, allowed))
    _close(process_logits(x, history, repetition=1.3, bias=bias[0], allowed=_bits(allowed)),
           *_reference(x, history, None, 1.3, 0.0, 0.0, bias[0], allowed))
    short = history.clamp(-1, V).int()
    _close(process_logits(x, short, lengths, presence=0.5, frequency=freq, allowed=_bits(allowed[-1])),
           *_reference(x, short, lengths, 1.0, 0.5, freq, None, allowed[-1]))
    _close(process_logits(x, allowed=allowed[-1]), *_reference(x, short[:, :0], None, 1.0, 0.0, 0.0, None, allowed[-1]))
    assert torch.equal(process_logits(x, history[:, :0], repetition=2.0), x)
    assert torch.equal(process_logits(x, history, lengths * 0, repetition=2.0), x)


def test_counts_of_one_token(cuda_device):
    """A history of one token many times over: the count is exact, whatever the order it was added up in."""
    from sparseforge_amd.logits import process_logits

    x = torch.zeros(1, 64, device=cuda_device)
    history = torch.full((1, 100003), 9, device=cuda_device)
    got = process_logits(x, history, frequency=1.0)
    assert got[0, 9] == -100003.0 and int((got != 0).sum()) == 1


def test_views_and_in_place(cuda_device):
    from sparseforge_amd.logits import process_logits

    g = torch.Generator(device=cuda_device).manual_seed(2)
    B, V = 3, 1003
    for dtype in (torch.bfloat16, torch.float32):
        every = torch.randn(B, 5, V, generator=g, device=cuda_device).to(dtype)
        history = torch.randint(0, V, (B, 64), generator=g, device=cuda_device)[:, ::2]  # strided ids
        bias = torch.randn(V, B, generator=g, device=cuda_device).T
        allowed = torch.rand(B, 2 * V, generator=g, device=cuda_device)[:, 1:V + 1] < 0.5
        last = every[:, -1]
        want = process_logits(last.contiguous(), history.contiguous(), repetition=1.5, bias=bias.contiguous(),
                              allowed=allowed.contiguous())
        assert torch.equal(process_logits(last, history, repetition=1.5, bias=bias, allowed=allowed), want)
        wide = torch.zeros(B, V + 9, dtype=dtype, device=cuda_device)
        got = process_logits(last, history, repetition=1.5, bias=bias, allowed=allowed, out=wide[:, 4:V + 4])
        assert torch.equal(got, want) and not wide[:, :4].any() and not wide[:, V + 4:].any()
        before = every[:, :4].clone()
        got = process_logits(last, history, repetition=1.5, bias=bias, allowed=allowed, out=last)
        assert got is last and torch.equal(every[:, -1], want) and torch.equal(every[:, :4], before)
        one = torch.randn(1, V, generator=g, device=cuda_device).to(dtype).expand(B, V)
        assert torch.equal(process_logits(one, history, presence=0.5),
                           process_logits(one.contiguous(), history, presence=0.5))


def test_values_that_are_not_finite(cuda_device):
    from sparseforge_amd.logits import process_logits

    x = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, math.nan, math.inf, 0.0, -0.0, 2.0]], device=cuda_device)
    history = torch.tensor([[0, 1, 2, 3]], device=cuda_device)
    allowed = torch.tensor([True] * 4 + [False] * 2 + [True] * 3, device=cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        got = process_logits(x.to(dtype), history, repetition=2.0, presence=1.0, allowed=allowed)[0]
        assert got[0].isnan() and got[1] == math.inf and got[2] == -math.inf and got[3] == -0.5
        assert got[4] == -math.inf and got[5] == -math.inf and got[8] == 2.0


def test_offsets_past_32_bits(cuda_device):
    """2.2e9 logits: the last rows are processed as rows of their own."""
    from sparseforge_amd.logits import process_logits

    B, V = 17000, 131072
    g = torch.Generator(device=cuda_device).manual_seed(4)
    row = torch.randn(1, V, generator=g, device=cuda_device).bfloat16()
    history = torch.randint(0, V, (B, 8), generator=g, device=cuda_device)
    freq = torch.rand(B, generator=g, device=cuda_device)
    got = process_logits(row.expand(B, V), history, frequency=freq)
    for b in (0, 16383, 16384, 16385, B - 1):
        assert torch.equal(got[b:b + 1], process_logits(row, history[b:b + 1], frequency=freq[b:b + 1].contiguous()))


def test_empty_and_refusals(cuda_device):
    from sparseforge_amd.logits import process_logits

    dev = cuda_device
    x = torch.zeros(2, 40, device=dev)
    ids = torch.zeros(2, 3, dtype=torch.int64, device=dev)
    assert process_logits(x[:0], ids[:0]).shape == (0, 40) and process_logits(x[:, :0], ids).shape == (2, 0)
    with pytest.raises(RuntimeError, match="GPU only"):
        process_logits(x.cpu())
    with pytest.raises(TypeError):
        process_logits(x.half())
    with pytest.raises(ValueError):
        process_logits(x[0])
    with pytest.raises(ValueError):
        process_logits(torch.zeros(65536, 2, device=dev))
    with pytest.raises(TypeError):
        process_logits(x, ids.float())
    for bad in (ids[:1], ids[0]):
        with pytest.raises(ValueError):
            process_logits(x, bad)
    for bad in (torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)):
        with pytest.raises(ValueError):
            process_logits(x, ids, bad)
    with pytest.raises(ValueError):
        process_logits(x, None, torch.zeros(2, dtype=torch.int32, device=dev))
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError):
            process_logits(x, ids, repetition=bad)
    for name in ("repetition", "presence", "frequency"):
        with pytest.raises(ValueError):
            process_logits(x, ids, **{name: torch.ones(3, device=dev)})
        with pytest.raises(RuntimeError):
            process_logits(x, ids, **{name: torch.ones(2)})
    with pytest.raises(TypeError):
        process_logits(x, bias=torch.zeros(40, dtype=torch.bfloat16, device=dev))
    with pytest.raises(ValueError):
        process_logits(x, bias=torch.zeros(39, device=dev))
    with pytest.raises(TypeError):
        process_logits(x, allowed=torch.ones(40, device=dev))
    for bad in (torch.ones(39, dtype=torch.bool, device=dev), torch.ones(2, 1, dtype=torch.int32, device=dev)):
        with pytest.raises(ValueError):
            process_logits(x, allowed=bad)
    for bad in (torch.empty(2, 39, device=dev), torch.empty(2, 40, dtype=torch.bfloat16, device=dev),
                torch.empty(40, 2, device=dev).T, torch.empty(1, 40, device=dev).expand(2, 40)):
        with pytest.raises(ValueError):
            process_logits(x, out=bad)
