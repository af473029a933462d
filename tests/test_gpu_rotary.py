"""rotary.rotary_embed (sf_rotary) against the turn of its pairs in float64.

Bars, per element with y = a c - b s (or b c + a s) from the float32 tables: two products and a sum in float32 are
off by at most 2^-24 of each product and of the sum, 2^-23 (|a c| + |b s|); storing in bf16 moves the result by half an
ulp more, 2^-8 |y|.  Copied elements are equal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _turn(x, cos, sin, positions, interleaved, inverse=False):
    """(y, sum of |terms|) in float64; positions [B, S], cos and sin [P, r / 2]."""
    x = x.double()
    c = cos.double()[positions][:, :, None]
    s = sin.double()[positions][:, :, None] * (-1.0 if inverse else 1.0)
    r = 2 * cos.shape[1]
    i0 = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    i1 = i0 + 1 if interleaved else i0 + r // 2
    i0, i1 = i0.to(x.device), i1.to(x.device)
    a, b = x[..., i0], x[..., i1]
    y, t = x.clone(), x.abs()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    t[..., i0], t[..., i1] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, t


def _check(got, x, cos, sin, positions, interleaved, inverse=False):
    assert got.is_contiguous() and got.dtype == x.dtype
    y, t = _turn(x, cos, sin, positions, interleaved, inverse)
    r = 2 * cos.shape[1]
    assert torch.equal(got[..., r:], x[..., r:])
    bar = t * 2.0 ** -23 + (y.abs() * 2.0 ** -8 if x.dtype == torch.bfloat16 else 0.0)
    assert bool(((got.double() - y).abs() <= bar).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hk,D,r", [(1, 1, 32, 32, 128, 128), (2, 65, 4, 2, 64, 64), (3, 7, 5, 1, 80, 20),
                                          (2, 33, 3, 3, 96, 24), (1, 130, 2, 1, 256, 64), (2, 5, 3, 2, 7, 2),
                                          (1, 9, 2, 2, 13, 12), (1, 3, 1, 1, 2, 2), (2, 17, 3, 1, 40, 36)])
def test_matches_float64(cuda_device, interleaved, dtype, B, S, H, Hk, D, r):
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    g = torch.Generator(device=cuda_device).manual_seed(S * 100 + D)
    q = torch.randn(B, S, H, D, generator=g, device=cuda_device).to(dtype)
    k = torch.randn(B, S, Hk, D, generator=g, device=cuda_device).to(dtype)
    cos, sin = rotary_cos_sin(300, r, device=cuda_device)
    plain = torch.arange(S, device=cuda_device).expand(B, S)
    drawn = torch.randint(0, 300, (B, S), generator=g, device=cuda_device)
    for given, positions in ((None, plain), (drawn, drawn), (drawn.int(), drawn), (drawn[0].int(), drawn[:1].expand(B, S))):
        got = rotary_embed(q, k, cos, sin, given, interleaved=interleaved)
        _check(got[0], q, cos, sin, positions, interleaved)
        _check(got[1], k, cos, sin, positions, interleaved)
    alone, none = rotary_embed(q, None, cos, sin, drawn, interleaved=interleaved)
    assert none is None and torch.equal(alone, rotary_embed(q, k, cos, sin, drawn, interleaved=interleaved)[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_inputs(cuda_device, interleaved):
    """Columns of a fused projection, an odd offset in memory, heads before tokens, a head that is not contiguous."""
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    g = torch.Generator(device=cuda_device).manual_seed(4)
    B, S, H, D = 2, 19, 4, 64
    cos, sin = rotary_cos_sin(S, D, device=cuda_device)
    at = torch.arange(S, device=cuda_device).expand(B, S)
    rows = torch.randn(B, S, 3 * H * D, generator=g, device=cuda_device).bfloat16()
    flat = torch.randn(B * S * H * D + 5, generator=g, device=cuda_device).bfloat16()
    forms = [rows[..., :H * D].view(B, S, H, D), rows[..., H * D:2 * H * D].view(B, S, H, D),
             flat[1:1 + B * S * H * D].view(B, S, H, D), flat[2:2 + B * S * H * D].view(B, S, H, D),
             flat[:B * S * H * D].view(B, H, S, D).transpose(1, 2), flat[:B * S * H * D].view(B, S, D, H).transpose(2, 3),
             rows[:, :1, :H * D].view(B, 1, H, D).expand(B, S, H, D)]
    for x in forms:
        for other in (forms[0], x):
            got = rotary_embed(other, x, cos, sin, interleaved=interleaved)
            _check(got[0], other, cos, sin, at, interleaved)
            _check(got[1], x, cos, sin, at, interleaved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(cuda_device, dtype, interleaved):
    from sparseforge_amd.rotary import RotaryScaling, rotary_cos_sin, rotary_embed

    g = torch.Generator(device=cuda_device).manual_seed(7)
    B, S, H, Hk, D, r = 2, 37, 6, 2, 80, 40
    cos, sin = rotary_cos_sin(128, r, scaling=RotaryScaling("yarn", 4.0, 32), device=cuda_device)
    positions = torch.randint(0, 128, (B, S), generator=g, device=cuda_device)
    rows = torch.randn(B, S, (H + Hk) * D, generator=g, device=cuda_device).to(dtype).requires_grad_(True)
    q, k = rows[..., :H * D].view(B, S, H, D), rows[..., H * D:].view(B, S, Hk, D)
    gq = torch.randn(B, S, H, D, generator=g, device=cuda_device).to(dtype)
    gk = torch.randn(B, S, 1, D, generator=g, device=cuda_device).to(dtype).expand(B, S, Hk, D)
    out = rotary_embed(q, k, cos, sin, positions, interleaved=interleaved)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True)
    _check(dq, gq, cos, sin, positions, interleaved, inverse=True)
    _check(dk, gk, cos, sin, positions, interleaved, inverse=True)
    # one output's gradient alone, and none for an input that takes none
    (only,) = torch.autograd.grad(out[1], k, gk, retain_graph=True)
    assert torch.equal(only, dk)
    kept = rotary_embed(q.detach(), k, cos, sin, positions, interleaved=interleaved)
    (only,) = torch.autograd.grad(kept[1], k, gk)
    assert torch.equal(only, dk)
    # through the fused projection's rows
    (drows,) = torch.autograd.grad(out, rows, (gq, gk), retain_graph=True)
    assert torch.equal(drows[..., :H * D].reshape(B, S, H, D), dq)
    # the derivative of the gradient along a direction: the turn again
    wq, wk = gq.clone().requires_grad_(True), torch.zeros_like(gk).requires_grad_(True)
    d = torch.autograd.grad(out, (q, k), (wq, wk), create_graph=True)
    (again,) = torch.autograd.grad(d[0], wq, gq)
    _check(again, gq, cos, sin, positions, interleaved)


def test_gradient_against_differences(cuda_device):
    """f(q) = <w, rotary(q)> is linear in q, so a difference over a step of any size is the gradient's product with it
    up to rounding: every output is off by at most 2^-23 (|a c| + |b s|) <= 2^-23 (|a| + |b|), |a|, |b| < 16."""
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    g = torch.Generator(device=cuda_device).manual_seed(8)
    cos, sin = rotary_cos_sin(50, 24, device=cuda_device)
    q = torch.randn(1, 50, 3, 32, generator=g, device=cuda_device).requires_grad_(True)
    w = torch.randn(1, 50, 3, 32, generator=g, device=cuda_device)
    step = torch.randn(1, 50, 3, 32, generator=g, device=cuda_device)
    for interleaved in (False, True):
        (dq,) = torch.autograd.grad(rotary_embed(q, None, cos, sin, interleaved=interleaved)[0], q, w)
        with torch.no_grad():
            far = rotary_embed(q + step, None, cos, sin, interleaved=interleaved)[0].double()
            near = rotary_embed(q - step, None, cos, sin, interleaved=interleaved)[0].double()
            moved = ((q + step).double() - (q - step).double())
        a = ((far - near) * w.double()).sum()
        b = (dq.double() * moved).sum()
        bar = 3 * 2.0 ** -23 * 32.0 * float(w.abs().sum() + moved.abs().sum())
        assert abs(float(a - b)) <= bar


def test_positions_outside_the_tables_give_nan(cuda_device):
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    cos, sin = rotary_cos_sin(10, 16, device=cuda_device)
    q = torch.ones(1, 4, 2, 24, device=cuda_device)
    positions = torch.tensor([[9, 10, -1, 0]], device=cuda_device)
    for given in (positions, positions.int()):
        for interleaved in (False, True):
            got = rotary_embed(q, None, cos, sin, given, interleaved=interleaved)[0]
            assert torch.equal(got[0, 1:3, :, :16].isnan().all(-1).all(-1), torch.tensor([True, True], device=cuda_device))
            assert not got[0, (0, 3)].isnan().any() and not got[..., 16:].isnan().any()


def test_more_than_one_launch_and_offsets_past_32_bits(cuda_device):
    """2.3e9 units of work and 3.5e9 elements: the last tokens are turned as the first ones."""
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    S, H, D = 1 << 20, 1100, 3
    g = torch.Generator(device=cuda_device).manual_seed(9)
    cos, sin = rotary_cos_sin(S, 2, device=cuda_device)
    row = torch.randn(1, 1, H, D, generator=g, device=cuda_device).bfloat16()
    got = rotary_embed(row.expand(1, S, H, D), None, cos, sin)[0]
    for at in (0, 1, (1 << 31) // (H * D) + 1, (1 << 31) // (2 * H), (1 << 31) // (2 * H) + 1, S - 1):
        _check(got[:, at:at + 1].contiguous(), row, cos, sin, torch.tensor([[at]], device=cuda_device), False)


def test_empty_and_refusals(cuda_device):
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    cos, sin = rotary_cos_sin(8, 16, device=cuda_device)
    q = torch.zeros(2, 4, 3, 16, device=cuda_device)
    assert rotary_embed(q[:, :0], q[:, :0], cos, sin)[0].shape == (2, 0, 3, 16)
    assert rotary_embed(q[:0], None, cos, sin)[0].shape == (0, 4, 3, 16)
    with pytest.raises(RuntimeError, match="GPU only"):
        rotary_embed(q.cpu(), None, cos, sin)
    with pytest.raises(TypeError):
        rotary_embed(q.half(), None, cos, sin)
    with pytest.raises(TypeError):
        rotary_embed(q, q.bfloat16(), cos, sin)
    with pytest.raises(TypeError):
        rotary_embed(q, None, cos.bfloat16(), sin)
    with pytest.raises(TypeError):
        rotary_embed(q, None, cos, sin, torch.zeros(2, 4, device=cuda_device))
    with pytest.raises(ValueError):
        rotary_embed(q, q[:, :3], cos, sin)
    with pytest.raises(ValueError):
        rotary_embed(q, None, cos, sin, torch.zeros(4, 2, dtype=torch.int32, device=cuda_device))
    with pytest.raises(ValueError):
        rotary_embed(q[..., :14], None, cos, sin)  # more pairs than the head has
    with pytest.raises(ValueError):
        rotary_embed(q.repeat(1, 3, 1, 1), None, cos, sin)  # 12 positions, 8 in the tables
    with pytest.raises(ValueError):
        rotary_embed(q, None, cos.requires_grad_(True), sin)
