"""distill.top_kl_loss with the rest, where a student's unlisted tokens hold next to nothing: losses that are finite have
finite gradients, that of the rest among them, which is f (P G - r) rho_j with rho the softmax over the unlisted tokens and G =
exp(Z_rest - Z).

Bars as in test_gpu_top_kl, with rho in the place of q: its exponent is off by 2^-24 (4 |a - Z_rest| + 8), the factors by dZ,
and dZ counts sums and entropies of float32 exponentials.  f rho (P G + r) E,  E = 2 dZ + 2^-24 (4 |a - Z_rest| + 8); along u
f / T rho ((P G + r) |u| + P G S + r S_r) (E + max E + dZ) with S = sum |u| q, S_r = sum |u| rho over the unlisted tokens.  The
listed tokens are formed in float64 with sums that are off by dZ: f (q + p) 2 dZ, along u f / T q (|u| + S) 2 dZ.

The definition is differentiated in float64 with the rest's log-sum-exp in two parts, its maximum and a logarithm: beside
-3.4e38, whose neighbours in float64 are 3.8e22 apart, the logarithm of a sum of 4000 is nothing.  Temperatures are float32.
"""
import math

import pytest
import torch
from test_gpu_sample import _f32
from test_gpu_top_kl import _inputs, _lse

pytestmark = pytest.mark.gpu


def _parts(s, t, lse, T):
    """Of rows [n, V] in float64: p by token, r, which are listed, log q, log rho (of unlisted tokens) and log G."""
    n, V = s.shape
    a = s.double() / T
    ids = t["ids"].reshape(n, -1).long()  # none of them is padding, or twice in a row
    listed = torch.zeros(n, V, dtype=torch.bool, device=s.device).scatter_(1, ids, True)
    entry = (t["values"].reshape(n, -1).double() / T - lse.reshape(n, 1).double()).exp()
    p = torch.zeros(n, V, dtype=torch.float64, device=s.device).scatter_(1, ids, entry)
    r = (1.0 - p.sum(-1, keepdim=True)).clamp_min(0.0)
    top = a.detach().amax(-1, keepdim=True)
    rest_top = a.detach().masked_fill(listed, -math.inf).amax(-1, keepdim=True)
    lz = (a - top).exp().sum(-1, keepdim=True).log()
    lzr = (a - rest_top).masked_fill(listed, -math.inf).exp().sum(-1, keepdim=True).log()
    return p, r, listed, (a - top) - lz, (a - rest_top) - lzr, (rest_top - top) + (lzr - lz)


def _loss(s, t, lse, T):
    p, r, listed, log_q, _, log_g = _parts(s, t, lse, T)
    kl = torch.where(listed, torch.special.xlogy(p, p) - p * log_q.masked_fill(~listed, 0.0), 0.0).sum(-1)
    kl = kl + torch.where(r > 0, r * (r.clamp_min(1e-300).log() - log_g), 0.0)[:, 0]
    w = t["weights"].double() if t["weights"] is not None else torch.ones_like(kl)
    return T * T * (w * kl).sum() / w.sum()


def check(t, T):
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    lse, s = _lse(t, T), t["s"].clone().requires_grad_(True)
    n, V = s.shape
    step = torch.finfo(s.dtype).eps / 2
    flat = s.detach().double().requires_grad_(True)
    want = _loss(flat, t, lse, T)
    g_want, = torch.autograd.grad(want, flat, create_graph=True)
    u = torch.randn(n, V, generator=t["g"], device=s.device).to(s.dtype)
    h_want, = torch.autograd.grad(g_want, flat, u.double())
    assert bool(want.isfinite()) and bool(g_want.isfinite().all()) and bool(h_want.isfinite().all())
    loss = top_kl_loss(s, TopLogits(t["values"], t["ids"], lse, T), T, weights=t["weights"])
    g, = torch.autograd.grad(loss, s, create_graph=True)
    h, = torch.autograd.grad(g, s, u)
    dZ = 2.0 ** -24 * (3 * (math.log(V) + 1) + 2 + V / 256 + 8)
    assert abs(loss.item() - want.item()) <= T * T * 2 * dZ + 2.0 ** -24 * abs(want.item())
    p, r, listed, log_q, d, log_g = _parts(s.detach(), t, lse, T)
    q, rho, G, P = log_q.exp(), d.masked_fill(listed, -math.inf).exp(), log_g.exp(), p.sum(-1, keepdim=True) + r
    w = t["weights"].double()[:, None] if t["weights"] is not None else torch.ones(n, 1, device=s.device).double()
    f = T * w / w.sum()
    E = 2 * dZ + 2.0 ** -24 * (4 * d.masked_fill(listed, 0.0).abs().clamp_max(800.0) + 8)
    U = u.double()
    S, Sr = (U.abs() * q).sum(-1, keepdim=True), (U.abs() * rho).sum(-1, keepdim=True)
    bar = torch.where(listed, f * (q + p) * 2 * dZ, f * rho * (P * G + r) * E)
    off = (g.detach().double() - g_want.detach()).abs()
    assert bool((off <= bar + step * g_want.detach().abs() + 1e-37).all()), float(off.max())
    bar = torch.where(listed, f / T * q * (U.abs() + S) * 2 * dZ,
                      f / T * rho * ((P * G + r) * U.abs() + P * G * S + r * Sr) * (E + E.amax(-1, keepdim=True) + dZ))
    off = (h.double() - h_want).abs()
    assert bool((off <= bar + step * h_want.abs() + 1e-37).all()), float(off.max())
    # it is the rest's gradient that is looked at: some of it is well above what rounds to nothing
    assert bool((g.detach().double().abs().masked_fill(listed | (w == 0), 0.0).amax(-1)[w[:, 0] != 0] > 1e-9).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gap", [40.0, 78.0, 85.0, 92.0, 110.0, 300.0, 800.0, 3.0e3, 1.0e5])
def test_unlisted_tokens_far_below(cuda_device, dtype, gap):
    """With few and with many rows (other numbers of threads), some of no weight."""
    for n, V, k in ((4, 5003, 16), (300, 515, 17)):
        t = _inputs(cuda_device, (n,), V, k, dtype, padded=False, weighted=n > 4)
        at = t["ids"].long()
        t["s"] = t["s"].scatter(1, at, (t["s"].gather(1, at).float() + gap).to(dtype))
        check(t, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_temperatures_below_1(cuda_device, dtype):
    """A confident row's gap of 30 is 120 at a temperature of 1/4 and 30000 at 1/1000."""
    for T in (0.25, 1e-3):
        t = _inputs(cuda_device, (4,), 3001, 12, dtype, padded=False, weighted=False)
        at = t["ids"].long()
        t["values"] = (t["values"].float() * T).to(dtype)
        t["s"] = (t["s"].float() * T).scatter(1, at, t["s"].gather(1, at).float() * T + 30.0).to(dtype)
        check(t, _f32(T))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-1e4, -1e9, None])
def test_unlisted_tokens_masked(cuda_device, dtype, low):
    """Every unlisted token at a mask's value: an equal share of the rest's gradient each."""
    t = _inputs(cuda_device, (3,), 4001, 9, dtype, padded=False, weighted=False)
    at = t["ids"].long()
    low = torch.finfo(dtype).min if low is None else low
    t["s"] = torch.full_like(t["s"], low).scatter(1, at, t["s"].gather(1, at))
    check(t, 1.0)


def test_rows_of_both_kinds_and_no_rest(cuda_device):
    """Rows with a rest near by, far below, and without one (the record's own sum), in one loss."""
    t = _inputs(cuda_device, (6,), 2050, 8, torch.float32, padded=False, weighted=False)
    at = t["ids"].long()
    shift = torch.tensor([0.0, 200.0, -200.0, 1000.0, 0.0, 50.0], device=cuda_device)[:, None]
    t["s"] = t["s"].scatter(1, at, t["s"].gather(1, at) + shift)
    check(t, 1.0)
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    lse = torch.logsumexp(t["values"].double(), -1).float() - 1e-3  # the listed tokens hold more than everything: r = 0
    s = t["s"].clone().requires_grad_(True)
    loss = top_kl_loss(s, TopLogits(t["values"], t["ids"], lse, 1.0), 1.0)
    g, = torch.autograd.grad(loss, s, create_graph=True)
    h, = torch.autograd.grad(g, s, torch.ones_like(s))
    flat = s.detach().double().requires_grad_(True)
    assert float(_parts(flat.detach(), t, lse, 1.0)[1].max()) == 0.0
    want = _loss(flat, t, lse, 1.0)
    w, = torch.autograd.grad(want, flat)
    assert abs(loss.item() - want.item()) <= 1e-5 + 1e-6 * abs(want.item())
    assert bool(((g.detach().double() - w).abs() <= 1e-5 * w.abs() + 1e-7).all()) and bool(h.isfinite().all())


def test_a_teacher_without_any_probability_shows(cuda_device):
    """A record of a row that is -inf throughout has a log-sum-exp of -inf: neither its entries nor the rest have a
    probability, and the loss and the row's gradient say so.  With a weight of 0 it is not looked at."""
    from sparseforge_amd.distill import top_kl_loss, top_logits

    g = torch.Generator(device=cuda_device).manual_seed(4)
    teacher = torch.randn(4, 500, generator=g, device=cuda_device)
    teacher[2] = -math.inf
    s = torch.randn(4, 500, generator=g, device=cuda_device, requires_grad=True)
    record = top_logits(teacher, 7)
    assert float(record.lse[2]) == -math.inf
    loss = top_kl_loss(s, record)
    assert not math.isfinite(loss.item())
    grad, = torch.autograd.grad(loss, s)
    assert not bool(grad[2].isfinite().any())
    weights = torch.tensor([1.0, 1.0, 0.0, 1.0], device=cuda_device)
    loss = top_kl_loss(s, record, weights=weights)
    grad, = torch.autograd.grad(loss, s)
    assert math.isfinite(loss.item()) and bool(grad.isfinite().all()) and bool((grad[2] == 0).all())


@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("entries", [1, 200])
def test_a_teachers_nan_shows(cuda_device, rest, entries):
    """Whichever entries of a row are NaN, all of them among these, or all that one part of the workgroup has."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    g = torch.Generator(device=cuda_device).manual_seed(5)
    s = torch.randn(3, 700, generator=g, device=cuda_device, requires_grad=True)
    ids = torch.rand(3, 700, generator=g, device=cuda_device).argsort(-1)[:, :entries].int()
    values = torch.randn(3, entries, generator=g, device=cuda_device)
    lse = torch.logsumexp(values, -1) + 0.1 if rest else None
    for part in (slice(None), slice(0, 64), slice(64, 128), slice(entries - 1, entries)):
        bad = values.clone()
        bad[1, part] = math.nan
        if not bool(bad.isnan().any()):
            continue
        loss = top_kl_loss(s, TopLogits(bad, ids, lse, 2.0 if rest else None))
        assert math.isnan(loss.item())
        grad, = torch.autograd.grad(loss, s)
        assert bool(grad[1].isnan().any()) and bool(grad[[0, 2]].isfinite().all())
    # entries of -inf have no probability, and without a log-sum-exp a row of nothing else adds nothing
    none = values.clone()
    none[1] = -math.inf
    if not rest:
        loss = top_kl_loss(s, TopLogits(none, ids))
        two = top_kl_loss(s[[0, 2]], TopLogits(values[[0, 2]], ids[[0, 2]]))
        assert abs(loss.item() - two.item() * 2 / 3) <= 1e-6 * two.item()
        assert bool((torch.autograd.grad(loss, s)[0][1] == 0).all())


def test_gradients_that_pass_the_caches(cuda_device):
    """More than 128 MB of them: four copies of 300 rows, whose listed tokens lie where float32 has no rho, have a fourth of
    these rows' gradients and products to the bit, the listed tokens' written over what came before."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (300,), 32000, 70, torch.float32, padded=False, weighted=False)
    at, lse = t["ids"].long(), _lse(t, 1.0)
    t["s"] = t["s"].scatter(1, at, t["s"].gather(1, at) + 150.0)
    u = torch.randn(300, 32000, generator=t["g"], device=cuda_device)
    seen = []
    for copies in (1, 4):
        s = t["s"].repeat(copies, 1).requires_grad_(True)
        teacher = TopLogits(t["values"].repeat(copies, 1), t["ids"].repeat(copies, 1), lse.repeat(copies), 1.0)
        g, = torch.autograd.grad(top_kl_loss(s, teacher, 1.0) * copies, s, create_graph=True)
        h, = torch.autograd.grad(g, s, u.repeat(copies, 1))
        seen.append((g.detach(), h))
    for one, four in zip(*seen):
        assert bool(one.isfinite().all()) and bool((one != 0).any())
        for part in four.split(300):
            assert torch.equal(part, one)
