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


def _sample(logits):
    """A pick that needs a distribution: multinomial refuses rows of NaN, which a softmax of -inf throughout gives."""
    p = logits.float().softmax(-1)
    assert not p.isnan().any()
    return torch.multinomial(p, 1)[:, 0]


@pytest.mark.parametrize("pick", [None, _sample])
def test_a_sequence_stops_where_nothing_may_follow(cuda_device, pick):
    """A grammar that counts up to a number of each sequence's own and is then complete, with and without a last token."""
    from sparseforge_amd.generate import generate

    m = _model(cuda_device)
    prompts = torch.tensor([[7, 10], [7, 20], [3, 30], [3, 500]], device=cuda_device)
    stop = torch.tensor([14, 20, 60, 502], device=cuda_device)
    ids = torch.arange(503, device=cuda_device)[None]

    def up(tokens, lengths):
        last = tokens.gather(1, lengths.long()[:, None] - 1)
        return (ids == last + 1) & (ids <= stop[:, None])

    tokens, ends = generate(m, prompts, 8, allowed=up, pick=pick)
    assert ends.tolist() == [6, 2, 10, 4]
    for row, n, first in zip(tokens.tolist(), ends.tolist(), (10, 20, 30, 500)):
        assert row[1:n] == list(range(first, first + n - 1))
    tokens, ends = generate(m, prompts, 8, allowed=up, pick=pick, end_token=13)
    assert ends.tolist() == [5, 2, 10, 4] and tokens[0, :5].tolist() == [7, 10, 11, 12, 13]
    none = torch.full((503,), float("-inf"), device=cuda_device)
    tokens, ends = generate(m, prompts, 3, bias=none, pick=pick)
    assert ends.tolist() == [2, 2, 2, 2] and torch.equal(tokens[:, :2], prompts)


@pytest.mark.parametrize("ragged", [False, True])
def test_a_captured_step_replayed(cuda_device, ragged):
    """One token a sequence as a graph, replayed over a block's edge with eager work and waits between the replays, each
    against the same step without a graph."""
    from sparseforge_amd.generate import Generator

    m = _model(cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(6)
    idx = torch.randint(0, 503, (2, 72), generator=g, device=cuda_device)
    plain, caught = Generator(m, 2, 80), Generator(m, 2, 80)
    for gen in (plain, caught):
        gen.step(idx[:, :60])
    now = torch.zeros(2, 1, dtype=torch.int64, device=cuda_device)
    counts = torch.ones(2, dtype=torch.int32, device=cuda_device) if ragged else None
    warm = Generator(m, 2, 80)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the kernels are loaded before the capture
        warm.step(now, counts)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    caught.cache.bound = 78
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = caught.step(now, counts)
    for i in range(60, 70):
        now.copy_(idx[:, i:i + 1])
        if ragged:
            counts[1] = i % 2
        plain.cache.bound = 78  # the same cut of the launch
        want = plain.step(now, counts)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) if not ragged or i % 2 else torch.equal(got[0], want[0])
        torch.randn(1000, device=cuda_device).sum().item()
    assert caught.cache.ends.tolist() == plain.cache.ends.tolist() == ([70, 65] if ragged else [70, 70])
