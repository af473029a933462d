"""Generator's attention against the model's own, which turns by its own tables and holds keys and values as they are.

A key's code is off by (largest of 64 tokens / 127) / sqrt(12) in the root of the mean square, 0.9 % of a normal key (its
largest is 4 times it), so scores of a spread of 2 are off by 0.02, the outputs, which are weighted by their exponentials,
by that much of their size, by 0.9 % more for the values and by 0.6 % for roundings to bf16: 3 % together.  The bar is three
times that; a rotation with other pairs, or off by one position, is an order of magnitude outside it."""
import pytest
import torch
from test_gpu_generate import _model, _Watched

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,steps", [(2, 64, [150]), (2, 64, [100, 1, 49]), (3, 128, [64, 1, 1, 84]),
                                             (2, 64, [1] * 70)])
def test_attention_is_the_models(cuda_device, heads, dim, steps):
    from sparseforge_amd.generate import Generator
    from sparseforge_amd.llama import causal_attention
    from sparseforge_amd.rotary import rotary_embed

    m = _model(cuda_device, heads, dim)
    m.init_random(torch.Generator(device=cuda_device).manual_seed(0), std=1.4 / (heads * dim) ** 0.5)  # scores of about 2
    watched = _Watched(m)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    S = sum(steps)
    idx = torch.randint(0, 503, (2, S), generator=g, device=cuda_device)
    gen = Generator(m, 2, S)
    seen, at = {}, 0
    for n in steps:
        gen.step(idx[:, at:at + n])
        at += n
        for key in [(i, name) for i in range(len(m.layers)) for name in "qkvo"]:
            seen.setdefault(key, []).append(watched.seen[key][0 if key[1] == "o" else 1].float())
    cos, sin = m._tables(S, cuda_device)
    for i in range(len(m.layers)):
        q, k, v, out = (torch.cat(seen[i, name], 1).view(2, S, heads, dim) for name in "qkvo")
        want = causal_attention(q, k, v, cos, sin).view(2, S, heads, dim)

        def off(x):
            return float((x - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt())

        assert off(out) < 0.09
        # other turns would show
        for wrong in (rotary_embed(q, k, gen.cos[:S], gen.sin[:S], interleaved=True),
                      (rotary_embed(q, None, gen.cos, gen.sin)[0], torch.roll(rotary_embed(k, None, gen.cos, gen.sin)[0], 1, 1))):
            none = torch.zeros_like(cos)
            assert off(causal_attention(*wrong, v, none + 1.0, none).view_as(want)) > 0.3
