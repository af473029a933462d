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
