"""rotary_embed where something other than a plain call looks in."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(cuda_device, grad):
    """An output without its tangent would be a derivative of 0."""
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    cos, sin = rotary_cos_sin(8, 16, device=cuda_device)
    q, k = (torch.randn(2, 4, 3, 16, device=cuda_device) for _ in range(2))
    with torch.set_grad_enabled(grad):
        want = rotary_embed(q, k, cos, sin)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(q, torch.ones_like(q))
            for args in ((dual, k), (k, dual), (dual, None)):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    rotary_embed(*args, cos, sin)
            got = rotary_embed(q, k, cos, sin)  # nothing to differentiate
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(lambda x: rotary_embed(x, k, cos, sin)[0], (q,), (torch.ones_like(q),))


def test_a_backward_notices_that_its_positions_have_moved_on(cuda_device):
    """The cache's starts as positions, and another step before the backward: its turn would be by the new positions."""
    from sparseforge_amd.kv_cache import KVCache8
    from sparseforge_amd.rotary import rotary_cos_sin, rotary_embed

    cos, sin = rotary_cos_sin(64, 16, device=cuda_device)
    cache = KVCache8(2, 1, 16, 64)
    cache.extend(5)
    cache.extend(1)
    q = torch.randn(2, 1, 3, 16, device=cuda_device, requires_grad=True)
    out = rotary_embed(q, None, cos, sin, cache.starts[:, None])[0]
    out.sum().backward(retain_graph=True)  # nothing has moved yet
    cache.extend(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with torch.inference_mode():
        own = KVCache8(2, 1, 16, 64)
        own.extend(5)
    own.extend(1)
    assert own.starts.tolist() == [5, 5] and own.ends.tolist() == [6, 6]
