"""What generate.generate and Generator.step do with inputs at their edges."""
import pytest
import torch
from test_gpu_generate import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [(0, 3), (4, -1), (5, 2), (1, 2 ** 31 - 1)])
def test_lengths_outside_the_prompts_are_refused(cuda_device, lengths):
    """A length past the prompts' columns would index past the tokens' rows; a row of none has nothing to continue."""
    from sparseforge_amd.generate import generate

    with pytest.raises(ValueError, match="lengths"):
        generate(_model(cuda_device), torch.zeros(2, 4, dtype=torch.int64, device=cuda_device), 3,
                 torch.tensor(lengths, dtype=torch.int32, device=cuda_device))


@pytest.mark.parametrize("chunk", [2048, 7])
def test_padding_may_be_any_id(cuda_device, chunk):
    """-1 and ids past the vocabulary beyond a row's length give what zeros there give."""
    from sparseforge_amd.generate import Generator, generate

    m = _model(cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(4)
    prompts = torch.randint(0, 503, (3, 20), generator=g, device=cuda_device)
    count = [20, 3, 9]
    lengths = torch.tensor(count, dtype=torch.int32, device=cuda_device)
    pad = torch.arange(20, device=cuda_device) >= lengths[:, None]
    got = {}
    for fill in (0, -1, -100, 503, 2 ** 40):
        tokens, ends = generate(m, prompts.masked_fill(pad, fill), 12, lengths, chunk=chunk, repetition=1.2)
        got[fill] = [row[:n].tolist() for row, n in zip(tokens, ends.tolist())]
        assert got[fill] == got[0] and [len(row) for row in got[fill]] == [n + 12 for n in count]
    for dtype in (torch.int32, torch.int64):
        a, b = (Generator(m, 3, 40).step(prompts.masked_fill(pad, fill).to(dtype), lengths) for fill in (0, -7))
        assert torch.equal(a, b)


def test_a_refused_step_leaves_the_cache_as_it_was(cuda_device):
    """Tokens of another batch, type or place are refused before the lengths advance, and the step may be taken again."""
    from sparseforge_amd.generate import Generator

    m = _model(cuda_device)
    idx = torch.arange(10, device=cuda_device).view(2, 5)
    want = Generator(m, 2, 64).step(idx)
    gen = Generator(m, 2, 64)
    for bad in (idx[:1], idx[0], idx.view(5, 2), idx.float(), idx.cpu(), idx[:, :0]):
        with pytest.raises(ValueError):
            gen.step(bad)
        assert gen.cache.bound == 0 and gen.cache.ends.tolist() == [0, 0]
    assert torch.equal(gen.step(idx), want)
