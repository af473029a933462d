"""generate() with a temperature: the draws are sample_logits' on the processed logits, with the generator's numbers."""
import pytest
import torch
from test_gpu_generate import _model

pytestmark = pytest.mark.gpu


def _prompts(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    return torch.randint(0, 503, (3, 9), generator=g, device=dev), torch.tensor([9, 4, 7], dtype=torch.int32, device=dev)


def test_draws_are_sample_logits(cuda_device):
    from sparseforge_amd.generate import generate
    from sparseforge_amd.logits import sample_logits

    m = _model(cuda_device)
    prompts, lengths = _prompts(cuda_device)
    settings = {"top_k": 40, "top_p": 0.9, "min_p": 0.01}
    seed = lambda: torch.Generator(device=cuda_device).manual_seed(7)  # noqa: E731
    got, ends = generate(m, prompts, 12, lengths, temperature=0.9, generator=seed(), repetition=1.2, end_token=5, **settings)
    g = seed()

    def pick(logits):
        return sample_logits(logits, torch.rand(3, device=cuda_device, generator=g), temperature=0.9, **settings)

    want, stops = generate(m, prompts, 12, lengths, pick=pick, repetition=1.2, end_token=5)
    assert torch.equal(ends, stops)
    for b in range(3):
        assert torch.equal(got[b, :ends[b]], want[b, :ends[b]])
    again, _ = generate(m, prompts, 12, lengths, temperature=0.9, generator=seed(), repetition=1.2, end_token=5, **settings)
    other, _ = generate(m, prompts, 12, lengths, temperature=0.9, generator=seed().manual_seed(8), repetition=1.2, **settings)
    assert torch.equal(got, again) and not torch.equal(got[:, :10], other[:, :10])


def test_temperature_0_is_the_most_likely_token(cuda_device):
    from sparseforge_amd.generate import generate

    m = _model(cuda_device)
    prompts, lengths = _prompts(cuda_device)
    got, ends = generate(m, prompts, 6, lengths, temperature=0.0)
    want, stops = generate(m, prompts, 6, lengths)
    assert torch.equal(ends, stops)
    for b in range(3):
        assert torch.equal(got[b, :ends[b]], want[b, :ends[b]])


def test_settings_of_each_sequence_and_masks(cuda_device):
    from sparseforge_amd.generate import generate

    m = _model(cuda_device)
    prompts, lengths = _prompts(cuda_device)
    allowed = torch.zeros(3, 503, dtype=torch.bool, device=cuda_device)
    allowed[0, 100:120] = True
    allowed[2, 33] = True  # sequence 1 may go on with nothing: it stops
    temperature = torch.tensor([1.5, 1.0, 0.0], device=cuda_device)
    top_k = torch.tensor([0, 3, 1], dtype=torch.int32, device=cuda_device)
    got, ends = generate(m, prompts, 5, lengths, temperature=temperature, top_k=top_k, allowed=allowed)
    assert ends.tolist() == [14, 4, 12]
    assert bool(((got[0, 9:14] >= 100) & (got[0, 9:14] < 120)).all()) and got[2, 7:12].tolist() == [33] * 5
    assert torch.equal(got[1, :4], prompts[1, :4])


def test_a_sequence_with_nan_logits_stops(cuda_device):
    """A NaN in one sequence's logits ends that sequence, and no id outside the vocabulary reaches the embedding."""
    from sparseforge_amd.generate import generate

    m = _model(cuda_device)
    prompts, lengths = _prompts(cuda_device)
    bias = torch.zeros(3, 503, device=cuda_device)
    bias[1, 17] = float("nan")
    got, ends = generate(m, prompts, 4, lengths, temperature=1.0, bias=bias)
    assert ends.tolist() == [13, 4, 11]
    assert bool(((got >= 0) & (got < 503)).all())


def test_refusals(cuda_device):
    from sparseforge_amd.generate import generate

    m = _model(cuda_device)
    prompts, _ = _prompts(cuda_device)
    with pytest.raises(ValueError):
        generate(m, prompts, 2, temperature=1.0, pick=lambda x: x.argmax(-1))
    for bad in ({"temperature": -1.0}, {"temperature": 1.0, "top_p": 2.0}, {"temperature": 1.0, "top_k": -1}):
        with pytest.raises(ValueError):
            generate(m, prompts, 2, **bad)


def test_settings_without_a_temperature_are_refused(cuda_device):
    from sparseforge_amd.generate import generate

    model, prompts = _model(cuda_device), torch.ones(2, 3, dtype=torch.int64, device=cuda_device)
    for bad in ({"top_k": 5}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_p": torch.ones(2, device=cuda_device)},
                {"generator": torch.Generator(device=cuda_device)}):
        with pytest.raises(ValueError, match="temperature"):
            generate(model, prompts, 2, **bad)
    generate(model, prompts, 2, top_k=0, top_p=1.0, min_p=0.0)
