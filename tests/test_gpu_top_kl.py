"""distill.top_kl_loss (sf_top_kl_*) against its definition in float64, differentiated by autograd, and differences.

Bars.  The row's Z = log sum exp(a), and that of the unlisted tokens, come from float32 exponentials: their arguments d = a
- max are off by 3 2^-24 |d|, |d| weighted by its share below ln V + 1; each rounds by 2^-23; a thread adds at most V /
256 + 8:
  dZ = 2^-24 (3 (ln V + 1) + 2 + V / 256 + 8)
The loss is P Z - r Z_r and float64 terms: at most T^2 2 dZ and 2^-24 of itself.  A gradient f q (P - r kappa): Z and
Z_r enter the factor in float64 (2 dZ), q's exponent is off by 2^-23 (|a - Z| + 2), the product rounds by 2^-23:
  f q (P + r kappa) E,  E = 2 dZ + 2^-23 (|a - Z| + 4)
The second derivative's product f q (A u - B) has the sums U and U_r in B, each off by E of its absolute sum and the
additions; its bar is f q ((P + r kappa) |u| + P S + r kappa^2 S_r) (E + dZ), S = sum |u| q.  Storing rounds by half a step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(dev, lead, V, k, dtype, seed=0, rest=True, padded=True, weighted=True, id_dtype=torch.int32, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed + V + k)
    n = math.prod(lead)
    ids = torch.rand(n, V, generator=g, device=dev).argsort(-1)[:, :k]
    values = (8.0 + torch.randn(n, k, generator=g, device=dev) * 2).to(dtype)
    s = torch.randn(n, V, generator=g, device=dev) * spread
    s.scatter_(1, ids, values.float() + torch.randn(n, k, generator=g, device=dev))
    if padded:
        length = torch.randint(0, k + 1, (n, 1), generator=g, device=dev)
        ids = ids.masked_fill(torch.arange(k, device=dev) >= length, -1)
        ids[0, 0] = V  # past the vocabulary: padding too
    weights = None
    if weighted:
        weights = torch.rand(n, generator=g, device=dev) + 0.1
        weights[::3] = 0.0
        weights = weights.view(lead)
    return {"s": s.to(dtype).view(*lead, V), "values": values.view(*lead, k), "ids": ids.to(id_dtype).view(*lead, k),
            "rest": rest, "weights": weights, "g": g}


def _lse(t, T):
    """A log-sum-exp over more than the listed tokens."""
    if not t["rest"]:
        return None
    V = t["s"].shape[-1]
    real = (t["ids"] >= 0) & (t["ids"] < V)
    b = (t["values"].double() / T).masked_fill(~real, -math.inf)
    n = torch.logsumexp(b, -1)
    more = -torch.log1p(-0.4 * torch.rand(n.shape, generator=t["g"], device=n.device, dtype=torch.float64))
    return torch.where(n.isfinite(), n + more, torch.zeros_like(n)).float()


def _rows(s, t, lse, T):
    """KL of every row in float64, differentiable in s (float64 [n, V])."""
    n, V = s.shape
    ids, b = t["ids"].reshape(n, -1).long(), t["values"].reshape(n, -1).double() / T
    real = (ids >= 0) & (ids < V)
    log_q = torch.log_softmax(s / T, -1)
    b = b.masked_fill(~real, -math.inf)
    norm = lse.reshape(n, 1).double() if lse is not None else torch.logsumexp(b, -1, keepdim=True)
    any_ = real.any(-1)
    log_p = torch.where(real, b - norm, 0.0)
    p = torch.where(real, log_p.exp(), 0.0)
    picked = torch.where(p > 0, log_q.gather(1, ids.clamp(0, V - 1)), 0.0)
    kl = torch.where(p > 0, p * (log_p.clamp_min(-1e300) - picked), 0.0).sum(-1)
    if lse is not None:
        flag = torch.zeros(n, V + 1, dtype=torch.bool, device=s.device)
        flag.scatter_(1, torch.where(real, ids, V), True)
        left = ~flag[:, :V]
        r = (1.0 - p.sum(-1)).clamp_min(0.0) * left.any(-1)
        rest = torch.logsumexp(log_q.masked_fill(~left, -math.inf), -1)
        kl = kl + torch.where(r > 0, r * (r.clamp_min(1e-300).log() - torch.where(r > 0, rest, 0.0)), 0.0)
    return torch.where(any_, kl, 0.0)


def _loss(s, t, lse, T):
    kl = _rows(s, t, lse, T)
    w = t["weights"].reshape(-1).double() if t["weights"] is not None else torch.ones_like(kl)
    total = w.sum()
    if float(total) == 0.0:
        return (kl * 0.0).sum()
    return T * T * torch.where(w != 0, w * kl, 0.0).sum() / total


def _bars(s, t, lse, T, scale, u):
    """Bars of the gradient and of the second derivative's product, from the module's formulas."""
    n, V = s.shape
    a = s.double() / T
    Z = torch.logsumexp(a, -1, keepdim=True)
    q = (a - Z).exp()
    dZ = 2.0 ** -24 * (3 * (math.log(V) + 1) + 2 + V / 256 + 8)
    E = 2 * dZ + 2.0 ** -23 * ((a - Z).abs().nan_to_num(posinf=0.0) + 4)
    rk = torch.zeros(n, 1, dtype=torch.float64, device=s.device)
    kappa = torch.zeros_like(rk)
    left = torch.ones(n, V, dtype=torch.bool, device=s.device)
    ids = t["ids"].reshape(n, -1).long()
    real = (ids >= 0) & (ids < V)
    if lse is not None:
        flag = torch.zeros(n, V + 1, dtype=torch.bool, device=s.device)
        flag.scatter_(1, torch.where(real, ids, V), True)
        left = ~flag[:, :V]
        p = torch.where(real, (t["values"].reshape(n, -1).double() / T - lse.reshape(n, 1).double()).exp(), 0.0)
        r = (1.0 - p.sum(-1, keepdim=True)).clamp_min(0.0) * left.any(-1, keepdim=True)
        Zr = torch.logsumexp(a.masked_fill(~left, -math.inf), -1, keepdim=True)
        kappa = torch.where(r > 0, (Z - Zr).exp(), 0.0)
        rk = r * kappa
    w = t["weights"].reshape(-1, 1).double() if t["weights"] is not None else torch.ones(n, 1, device=s.device).double()
    f = torch.where(w != 0, scale * T * w / w.sum(), 0.0)
    grad = f * q * (1.0 + rk) * E
    if u is None:
        return grad, None
    S = (u.abs() * q).sum(-1, keepdim=True)
    Sr = (u.abs() * q * left).sum(-1, keepdim=True)
    second = f / T * q * ((1.0 + rk) * u.abs() + S + rk * kappa * Sr) * (E + E.amax(-1, keepdim=True) + dZ)
    return grad, second


def check(t, T, scale=1.0, hvp=True):
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    s, lse = t["s"], _lse(t, T)
    V = s.shape[-1]
    n = s.numel() // V
    step = torch.finfo(s.dtype).eps / 2
    mine = s.detach()
    mine.requires_grad_(True)
    loss = top_kl_loss(mine, TopLogits(t["values"], t["ids"], lse, T), T, weights=t["weights"])
    assert loss.dtype == torch.float32 and loss.shape == ()
    flat = s.detach().reshape(n, V).double().requires_grad_(True)
    want = _loss(flat, t, lse, T)
    dZ = 2.0 ** -24 * (3 * (math.log(V) + 1) + 2 + V / 256 + 8)
    assert abs(loss.item() - want.item()) <= T * T * 2 * dZ + 2.0 ** -24 * abs(want.item())
    u = torch.randn(n, V, generator=t["g"], device=s.device).to(s.dtype)
    g_want, = torch.autograd.grad(want * scale, flat, create_graph=hvp)
    g, = torch.autograd.grad(loss * scale, mine, create_graph=hvp)
    assert g.dtype == s.dtype and g.shape == s.shape
    g_bar, h_bar = _bars(s.detach().reshape(n, V), t, lse, T, scale, u.double() if hvp else None)
    diff = (g.detach().reshape(n, V).double() - g_want.detach()).abs()
    assert bool((diff <= g_bar + step * g_want.detach().abs() + 1e-37).all()), float(diff.max())
    if hvp:
        h_want, = torch.autograd.grad(g_want, flat, u.double())
        h, = torch.autograd.grad(g, mine, u.view(s.shape))
        assert h.dtype == s.dtype
        diff = (h.reshape(n, V).double() - h_want).abs()
        assert bool((diff <= h_bar + step * h_want.abs() + 1e-37).all()), float(diff.max())
    return loss


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("lead,V,k", [((1,), 2, 1), ((3,), 7, 3), ((2, 5), 33, 8), ((4,), 1001, 1), ((3,), 2050, 300),
                                      ((2, 3), 32000, 64), ((2,), 50257, 20), ((2,), 131072, 1000), ((300,), 515, 17)])
def test_matches_float64(cuda_device, dtype, rest, lead, V, k):
    for T, padded, weighted, id_dtype in ((2.0, False, False, torch.int32), (1.0, True, True, torch.int64)):
        t = _inputs(cuda_device, lead, V, k, dtype, rest=rest, padded=padded, weighted=weighted, id_dtype=id_dtype)
        check(t, T, scale=0.25 if padded else 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rest", [True, False])
def test_every_token_listed(cuda_device, dtype, rest):
    """With nothing left the other tokens have no share, whatever the log-sum-exp's rounding says."""
    check(_inputs(cuda_device, (4,), 40, 40, dtype, rest=rest, padded=False), 2.0)


@pytest.mark.parametrize("rest", [True, False])
def test_an_id_listed_twice_counts_twice(cuda_device, rest):
    for dtype, k in ((torch.bfloat16, 12), (torch.float32, 600)):
        t = _inputs(cuda_device, (5,), 3001, k, dtype, rest=rest, padded=False)
        t["ids"][0, 3] = t["ids"][0, 0]
        t["ids"][0, k - 1] = t["ids"][0, 0]
        t["ids"][2] = t["ids"][2, 0]
        t["ids"][4, 1] = t["ids"][4, k - 2]
        check(t, 2.0)


def test_other_value_type(cuda_device):
    t = _inputs(cuda_device, (6,), 999, 9, torch.bfloat16)
    t["values"] = t["values"].float() + 0.003
    check(t, 1.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_students(cuda_device, dtype):
    """A shifted view, a slice of columns (odd addresses), an expanded and a transposed student; a gradient that is not
    contiguous."""
    t = _inputs(cuda_device, (3, 6), 1003, 9, dtype)
    full = t["s"].clone()
    t["s"] = full[:, :-1]
    for name in ("values", "ids", "weights"):
        t[name] = t[name][:, :-1]
    check(t, 2.0)
    t = _inputs(cuda_device, (4,), 1003, 9, dtype)
    wide = torch.zeros(4, 1100, device=cuda_device, dtype=dtype)
    wide[:, 5:1008] = t["s"]
    t["s"] = wide[:, 5:1008]
    check(t, 2.0)
    t["s"] = t["s"][:1].expand(4, 1003)
    check(t, 2.0)
    t["s"] = t["s"].t().contiguous().t()
    check(t, 2.0)


def test_distribution_far_apart(cuda_device):
    """Students whose listed or unlisted tokens hold almost nothing."""
    for shift in (30.0, -30.0):
        t = _inputs(cuda_device, (4,), 5000, 16, torch.float32, padded=False, spread=4.0)
        t["s"].scatter_add_(1, t["ids"].long(), torch.full((4, 16), shift, device=cuda_device))
        # the rest's share of 1e-13 divides the gradient of its own tokens: kappa is in the bars
        check(t, 1.0)


def test_rows_that_do_not_count(cuda_device):
    """Rows of weight 0 may hold anything; rows without entries add nothing; no weight at all gives 0."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    for rest in (True, False):
        t = _inputs(cuda_device, (6,), 700, 5, torch.float32, rest=rest, padded=False, weighted=False)
        lse = _lse(t, 2.0)
        t["weights"] = torch.tensor([1.0, 0.0, 2.0, 0.0, 1.0, 1.0], device=cuda_device)
        t["ids"][4] = -1
        s = t["s"].clone()
        s[1] = math.nan
        s[3, 5] = math.inf
        s[4] = math.nan  # no entries: not looked at either
        t["values"][3] = math.nan
        s.requires_grad_(True)
        loss = top_kl_loss(s, TopLogits(t["values"], t["ids"], lse, 2.0), weights=t["weights"])
        g, = torch.autograd.grad(loss, s, create_graph=True)
        h, = torch.autograd.grad(g, s, torch.ones_like(g))
        ok = [0, 2, 5]
        kl = _rows(s.detach()[ok].double(), {"ids": t["ids"][ok], "values": t["values"][ok]},
                   lse[ok] if rest else None, 2.0)
        want = 4.0 * (kl * torch.tensor([1.0, 2.0, 1.0], device=cuda_device)).sum() / 5.0
        assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
        for y in (g, h):
            assert bool((y[[1, 3, 4]] == 0).all()) and bool(y[ok].isfinite().all()) and bool((y[ok] != 0).any())
        none = top_kl_loss(s, TopLogits(t["values"], t["ids"], lse), weights=torch.zeros(6, device=cuda_device))
        assert float(none) == 0.0
        assert bool((torch.autograd.grad(none, s)[0] == 0).all())
    empty = torch.zeros(0, 50, device=cuda_device, requires_grad=True)
    loss = top_kl_loss(empty, TopLogits(torch.zeros(0, 3, device=cuda_device),
                                        torch.zeros(0, 3, device=cuda_device, dtype=torch.int32)))
    assert float(loss) == 0.0 and torch.autograd.grad(loss, empty)[0].shape == (0, 50)


def test_what_is_not_finite_shows(cuda_device):
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (2,), 300, 4, torch.float32, padded=False, weighted=False)
    teacher = TopLogits(t["values"], t["ids"])
    s = t["s"].clone()
    s[0, t["ids"][0, 1].long()] = -math.inf  # a token that the teacher wants has no probability
    assert float(top_kl_loss(s, teacher)) == math.inf
    s[0, 3] = math.nan
    assert math.isnan(float(top_kl_loss(s, teacher)))
    s = t["s"].clone()
    s[:, 17:29] = -math.inf  # tokens that the teacher does not ask for
    s[0, t["ids"][0].long()] = t["s"][0, t["ids"][0].long()]
    s[1, t["ids"][1].long()] = t["s"][1, t["ids"][1].long()]
    t["s"], t["rest"], t["weights"] = s, False, None
    check(t, 2.0)
    t["rest"] = True
    check(t, 2.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rest", [True, False])
def test_tokens_masked_by_the_lowest_value(cuda_device, dtype, rest):
    """The type's lowest value in place of -inf: tokens of no probability among others, equal tokens alone."""
    t = _inputs(cuda_device, (4,), 777, 6, dtype, rest=rest, padded=False, weighted=False)
    lowest = torch.finfo(dtype).min
    keep = t["s"].clone()
    t["s"][1, 100:700] = lowest
    t["s"][1] = torch.where(torch.zeros(777, dtype=torch.bool, device=cuda_device)
                            .index_fill_(0, t["ids"][1].long(), True), keep[1], t["s"][1])
    t["s"][2] = lowest
    check(t, 2.0, hvp=False)


def test_agrees_with_the_whole_teacher(cuda_device):
    """With every token recorded the loss is chunked_kl_loss'."""
    from sparseforge_amd.distill import chunked_kl_loss, top_kl_loss, top_logits

    g = torch.Generator(device=cuda_device).manual_seed(1)
    s, t = (torch.randn(12, 1000, generator=g, device=cuda_device) * 3 for _ in range(2))
    whole = chunked_kl_loss(s, t)
    for top in (top_logits(t, 1000), top_logits(t, 1000)._replace(lse=None)):
        assert abs(float(top_kl_loss(s, top)) - float(whole)) <= 2e-6 * float(whole) + 1e-5
    # and a cross-entropy where the one entry is certain
    ids = torch.randint(0, 1000, (12, 1), generator=g, device=cuda_device)
    from sparseforge_amd.distill import TopLogits

    one = top_kl_loss(s, TopLogits(torch.zeros(12, 1, device=cuda_device), ids), 1.0)
    want = torch.nn.functional.cross_entropy(s.double(), ids[:, 0])
    assert abs(float(one) - float(want)) <= 1e-6 * float(want) + 1e-5


def test_gradient_against_differences(cuda_device):
    """Central differences of the loss itself: of step e, off by e^2 / 6 times a third derivative below T^2 / T^3, and by
    the loss' rounding 2 2^-24 |loss| and dZ over 2 e."""
    t = _inputs(cuda_device, (2,), 60, 6, torch.float32, padded=False, weighted=False)
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    T = 2.0
    teacher = TopLogits(t["values"], t["ids"], _lse(t, T), T)
    s = t["s"].clone().requires_grad_(True)
    loss = top_kl_loss(s, teacher, T)
    g, = torch.autograd.grad(loss, s)
    e = 2.0 ** -5
    with torch.no_grad():
        for i, j in ((0, 0), (1, 59), (0, int(t["ids"][0, 0])), (1, int(t["ids"][1, 3]))):
            d = torch.zeros_like(s)
            d[i, j] = e
            slope = (float(top_kl_loss(s + d, teacher, T)) - float(top_kl_loss(s - d, teacher, T))) / (2 * e)
            noise = (2.0 ** -24 * 2 * abs(float(loss)) + T * T * 2 * 2.0 ** -24 * 40) / e
            assert abs(slope - float(g[i, j])) <= e * e / T + noise


def test_gradient_of_the_upstream_factor(cuda_device):
    """c * loss differentiated twice where c is a leaf: the factor's gradient is the direction's product."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (5,), 400, 7, torch.float32)
    lse = _lse(t, 2.0)
    s = t["s"].clone().requires_grad_(True)
    c = torch.tensor(0.5, device=cuda_device, requires_grad=True)
    g, = torch.autograd.grad(c * top_kl_loss(s, TopLogits(t["values"], t["ids"], lse, 2.0), weights=t["weights"]), s,
                             create_graph=True)
    u = torch.randn(s.shape, generator=t["g"], device=cuda_device)
    gc, h = torch.autograd.grad(g, (c, s), u)
    flat = s.detach().double().requires_grad_(True)
    want_g, = torch.autograd.grad(_loss(flat, t, lse, 2.0), flat)
    dot = float((want_g * u.double()).sum())
    assert abs(float(gc) - dot) <= 1e-5 * float((want_g * u.double()).abs().sum())
    assert bool(h.isfinite().all())


def test_refusals(cuda_device):
    from sparseforge_amd.distill import TopLogits, top_kl_loss, top_logits

    t = _inputs(cuda_device, (2, 3), 50, 4, torch.float32)
    s, v, i = t["s"], t["values"], t["ids"]
    lse = torch.zeros(2, 3, device=cuda_device)
    for teacher, T in ((TopLogits(v[:1], i[:1]), 2.0), (TopLogits(v, i[..., :3]), 2.0), (TopLogits(v, i, lse[0]), 2.0),
                       (TopLogits(v, i, lse.double()), 2.0), (TopLogits(v, i, lse, 1.0), 2.0), (TopLogits(v, i), 0.0),
                       (TopLogits(v, i), math.nan), (TopLogits(v, i), math.inf)):
        with pytest.raises(ValueError):
            top_kl_loss(s, teacher, T)
    with pytest.raises(TypeError):
        top_kl_loss(s, TopLogits(v, i.float()))
    with pytest.raises(TypeError):
        top_kl_loss(s.half(), TopLogits(v, i))
    with pytest.raises(TypeError):
        top_kl_loss(s, TopLogits(v.double(), i))
    with pytest.raises(ValueError):
        top_kl_loss(s, TopLogits(v, i), weights=torch.ones(6, device=cuda_device))
    with pytest.raises(RuntimeError):
        top_kl_loss(s, TopLogits(v.cpu(), i))
    with pytest.raises(ValueError):
        top_kl_loss(s, top_logits(s, 4, 1.0), 2.0)


def test_captured_step(cuda_device):
    """Forward and backward captured into a graph and replayed on new logits."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (4,), 32000, 64, torch.bfloat16, weighted=False, padded=False)
    teacher = TopLogits(t["values"], t["ids"], _lse(t, 2.0), 2.0)
    s = t["s"].clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(top_kl_loss(s, teacher), s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = top_kl_loss(s, teacher)
        g, = torch.autograd.grad(loss, s)
        loss = loss.detach()
    for _ in range(3):
        with torch.no_grad():
            s.copy_(torch.randn(s.shape, generator=t["g"], device=cuda_device) * 2)
        graph.replay()
        torch.cuda.synchronize()
        again = top_kl_loss(s, teacher)
        assert float(loss) == float(again)
        assert torch.equal(g, torch.autograd.grad(again, s)[0])


def test_results_do_not_vary(cuda_device):
    t = _inputs(cuda_device, (64,), 5001, 33, torch.bfloat16)
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    lse = _lse(t, 2.0)
    s = t["s"].requires_grad_(True)
    first = None
    for _ in range(3):
        loss = top_kl_loss(s, TopLogits(t["values"], t["ids"], lse), weights=t["weights"])
        g, = torch.autograd.grad(loss, s)
        if first is None:
            first = loss.detach(), g
        assert torch.equal(first[0], loss.detach()) and torch.equal(first[1], g)


def test_plain_and_recorded_backward_agree(cuda_device):
    """A plain backward pass and one that records give the same gradients; forward mode and vmap are refused, not passed
    by."""
    from torch.autograd import forward_ad

    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (7,), 300, 5, torch.float32)
    teacher = TopLogits(t["values"], t["ids"], _lse(t, 2.0), 2.0)
    s = t["s"].requires_grad_(True)
    loss = top_kl_loss(s, teacher, weights=t["weights"])
    a, = torch.autograd.grad(loss, s, retain_graph=True)
    b, = torch.autograd.grad(loss, s, create_graph=True)
    assert b.requires_grad and not a.requires_grad and torch.equal(a, b.detach())
    with torch.no_grad():
        assert torch.equal(loss.detach(), top_kl_loss(s, teacher, weights=t["weights"]))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(s.detach(), torch.ones_like(s))
        with pytest.raises(NotImplementedError):
            top_kl_loss(dual, teacher, weights=t["weights"])
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: top_kl_loss(x, teacher))(s.detach()[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: top_kl_loss(x, teacher))(s.detach())


def test_rows_of_no_weight_beside_a_weight_that_is_nan(cuda_device):
    """A NaN among the weights shows in the rows that count; rows of weight 0 still take zeros."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (4,), 900, 6, torch.float32, padded=False, weighted=False)
    weights = torch.tensor([1.0, 0.0, math.nan, 0.0], device=cuda_device)
    s = t["s"].requires_grad_(True)
    loss = top_kl_loss(s, TopLogits(t["values"], t["ids"], _lse(t, 2.0), 2.0), weights=weights)
    g, = torch.autograd.grad(loss, s, create_graph=True)
    h, = torch.autograd.grad(g, s, torch.ones_like(g))
    for y in (g, h):
        assert bool((y[[1, 3]] == 0).all()) and bool(y[[0, 2]].isnan().any(-1).all())


def test_shapes_that_are_refused(cuda_device):
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    v, i = torch.zeros(2, 5000, device=cuda_device), torch.zeros(2, 5000, dtype=torch.int32, device=cuda_device)
    with pytest.raises(ValueError):
        top_kl_loss(torch.zeros(2, 6000, device=cuda_device), TopLogits(v, i))  # too many entries
    with pytest.raises(ValueError):
        top_kl_loss(torch.zeros(2, 0, device=cuda_device), TopLogits(v[:, :0], i[:, :0]))
    with pytest.raises(ValueError):
        top_kl_loss(torch.zeros((), device=cuda_device), TopLogits(v[0, :1], i[0, :1]))
    # no entries at all: nothing to learn
    s = torch.randn(2, 30, device=cuda_device, requires_grad=True)
    loss = top_kl_loss(s, TopLogits(v[:, :0], i[:, :0], torch.zeros(2, device=cuda_device), 2.0))
    assert float(loss) == 0.0 and bool((torch.autograd.grad(loss, s)[0] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_behind_2_31_elements(cuda_device, dtype):
    """The last rows of logits whose offsets pass 32 bits, with their gradient and second derivative."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    B, V, k = 8300, 262144 if dtype == torch.bfloat16 else 262143, 12
    t = _inputs(cuda_device, (3,), V, k, dtype, padded=False, weighted=False)
    lse = _lse(t, 2.0)
    s = torch.zeros(B, V, dtype=dtype, device=cuda_device)
    s[-3:] = t["s"]
    ids = torch.full((B, k), -1, dtype=torch.int32, device=cuda_device)
    values, all_lse = torch.zeros(B, k, dtype=dtype, device=cuda_device), torch.zeros(B, device=cuda_device)
    weights = torch.zeros(B, device=cuda_device)
    ids[-3:], values[-3:], all_lse[-3:], weights[-3:] = t["ids"], t["values"], lse, 1.0
    weights[5] = 1.0  # counts, without entries
    u = torch.zeros_like(s)
    u[-3:] = torch.randn(3, V, generator=t["g"], device=cuda_device).to(dtype)
    s.requires_grad_(True)
    loss = top_kl_loss(s, TopLogits(values, ids, all_lse, 2.0), weights=weights)
    g, = torch.autograd.grad(loss, s, create_graph=True)
    h, = torch.autograd.grad(g, s, u)
    few = torch.cat([s.detach()[5:6], s.detach()[-3:]]).requires_grad_(True)
    pick = [5, B - 3, B - 2, B - 1]
    alone = top_kl_loss(few, TopLogits(values[pick], ids[pick], all_lse[pick], 2.0))
    g1, = torch.autograd.grad(alone, few, create_graph=True)
    h1, = torch.autograd.grad(g1, few, u[pick])
    # other threads to a row: the sums of float32 exponentials differ in their order
    bar = 2.0 ** -23 * (3 * (math.log(V) + 1) + 10 + V / 256) * 4
    assert abs(float(loss.detach()) - float(alone.detach())) <= 4 * bar
    for big, small in ((g.detach(), g1.detach()), (h, h1)):
        step = torch.finfo(dtype).eps
        near = (big[-3:].double() - small[1:].double()).abs()
        assert bool((near <= (bar + step) * small[1:].double().abs() + bar * small.double().abs().amax(-1)[1:, None]).all())
        for part in big[:-3].split(1000):
            assert not bool((part != 0).any())


def test_record_then_distil(cuda_device):
    """top_logits' record of a teacher, kept in float32 or as it is, and the loss from it, against the definition; on a
    stream of its own beside another."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss, top_logits

    g = torch.Generator(device=cuda_device).manual_seed(21)
    teacher = (torch.randn(2, 9, 32000, generator=g, device=cuda_device) * 3).bfloat16()
    student = (teacher.float() + torch.randn(2, 9, 32000, generator=g, device=cuda_device)).bfloat16()
    for k in (1, 50, 1000):
        record = top_logits(teacher, k, 1.5)
        t = {"s": student.clone(), "values": record.values, "ids": record.ids, "weights": None}
        want = _loss(student.view(18, -1).double(), t, record.lse, 1.5)
        dZ = 2.0 ** -24 * (3 * (math.log(32000) + 1) + 2 + 32000 / 256 + 8)
        for values in (record.values, record.values.float()):
            kept = TopLogits(values, record.ids.long(), record.lse, 1.5)
            got = top_kl_loss(student, kept, 1.5)
            assert abs(float(got) - float(want)) <= 1.5 ** 2 * 2 * dZ + 2.0 ** -24 * abs(float(want))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        outs = []
        for stream in streams * 3:
            with torch.cuda.stream(stream):
                outs.append(top_kl_loss(student, top_logits(teacher, k, 1.5), 1.5))
        torch.cuda.synchronize()
        assert all(float(o) == float(outs[0]) for o in outs)


def test_captured_second_derivative(cuda_device):
    """Loss, gradient and the second derivative's product in one graph, beside another graph of the same tensors, replayed in
    turn on new logits and weights with eager work between."""
    from sparseforge_amd.distill import TopLogits, top_kl_loss

    t = _inputs(cuda_device, (6,), 5001, 30, torch.float32, padded=False)
    teacher = TopLogits(t["values"], t["ids"], _lse(t, 2.0), 2.0)
    s, weights = t["s"].clone().requires_grad_(True), t["weights"].clone()
    u = torch.randn(s.shape, generator=t["g"], device=cuda_device)

    def step():
        loss = top_kl_loss(s, teacher, weights=weights)
        g, = torch.autograd.grad(loss, s, create_graph=True)
        h, = torch.autograd.grad(g, s, u)
        return loss.detach(), g.detach(), h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for _ in range(3):
        with torch.no_grad():
            s.copy_(torch.randn(s.shape, generator=t["g"], device=cuda_device) * 2)
            weights.copy_(torch.rand(weights.shape, generator=t["g"], device=cuda_device))
            weights[2] = 0.0
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_next_to_the_row_are_left(cuda_device, dtype):
    """Gradients are written to their rows alone, whatever the alignment: rows of odd lengths beside others."""
    from sparseforge_amd import _lib as L
    from sparseforge_amd.distill_top import _top_kl_desc, _top_kl_forward

    for V in (1, 7, 8, 9, 130, 4099):
        t = _inputs(cuda_device, (5,), V, 1, dtype, padded=False, weighted=False)
        lse = _lse(t, 2.0)
        ids = t["ids"].contiguous()
        loss, state = _top_kl_forward(t["s"], t["values"], ids, lse, None, 2.0)
        one = torch.ones((), device=cuda_device)
        guard = torch.full((5 * V + 64,), 7.0, dtype=dtype, device=cuda_device)
        desc, keep = _top_kl_desc(t["s"], t["values"], ids, lse, None, state, 2.0)
        for at in (0, 1, 8, 13):
            guard.fill_(7.0)
            out = guard[32 + at:32 + at + 5 * V]
            L.check(L.lib().sf_top_kl_backward(desc, one.data_ptr(), out.data_ptr(), L.stream(t["s"].device)), "backward")
            assert bool((guard[:32 + at] == 7.0).all()) and bool((guard[32 + at + 5 * V:] == 7.0).all())
            assert bool(out.isfinite().all()) and not bool((out == 7.0).any())
