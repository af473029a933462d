"""process_logits with an `out` that something else knows of."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_backward_notices_that_its_saved_result_was_written(cuda_device):
    from sparseforge_amd.logits import process_logits

    x = torch.randn(2, 50, device=cuda_device, requires_grad=True)
    history = torch.zeros(2, 3, dtype=torch.int64, device=cuda_device)
    lp = x.log_softmax(-1)
    with torch.no_grad():
        process_logits(lp, history, presence=1.0, out=lp)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()
    # a view of it, and one that is only read
    lp = x.log_softmax(-1)
    rows = lp.detach()
    before = rows._version
    process_logits(rows, history, presence=1.0)
    assert rows._version == before
    process_logits(rows[:1], history[:1], presence=1.0, out=rows[1:])
    assert rows._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()


def test_an_out_that_requires_grad(cuda_device):
    from sparseforge_amd.logits import process_logits

    x = torch.randn(2, 50, device=cuda_device)
    out = torch.zeros(2, 50, device=cuda_device, requires_grad=True)
    with pytest.raises(ValueError, match="requires grad"):
        process_logits(x, out=out)
    with torch.no_grad():  # as torch's own in-place operations
        assert torch.equal(process_logits(x, out=out), x)
    with torch.inference_mode():
        own = torch.empty_like(x)
        process_logits(x, out=own)
    assert process_logits(x, out=own) is own


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_an_out_that_lies_over_the_logits(cuda_device, dtype):
    """Rows written where other rows are still to be read: shifted by a row, by a few elements, of another stride, of one
    row for all; and the forms that share memory without sharing an element."""
    from sparseforge_amd.logits import process_logits

    g = torch.Generator(device=cuda_device).manual_seed(8)
    B, V = 300, 20001
    history = torch.randint(0, V, (B, 9), generator=g, device=cuda_device)
    data = torch.randn((B + 1) * (V + 7) * 2, generator=g, device=cuda_device).to(dtype)

    def rows(first, stride):
        return lambda t: t.as_strided((B, V), (stride, 1), first)

    for x, y in ((rows(0, V), rows(V, V)), (rows(V, V), rows(0, V)), (rows(0, V), rows(3, V)), (rows(5, V), rows(0, V)),
                 (rows(0, V + 7), rows(1, V)), (rows(0, V), rows(2, V + 7)), (rows(V, 0), rows(0, V)),
                 (rows(0, 2 * V), rows(V, 2 * V)), (rows(V, 2 * V), rows(0, 2 * V)), (rows(0, V), rows(0, V)),
                 (rows(0, 2 * V), rows(V - 1, 2 * V))):
        want = process_logits(x(data).clone(), history, presence=0.5, frequency=0.25)
        t = data.clone()
        got = process_logits(x(t), history, presence=0.5, frequency=0.25, out=y(t))
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B", [100, 300, 600])
def test_rows_do_not_depend_on_how_many_there_are(cuda_device, dtype, B):
    """Outputs on both sides of what is written past the caches: each row as it is alone."""
    from sparseforge_amd.logits import process_logits

    g = torch.Generator(device=cuda_device).manual_seed(B)
    V = 131072
    x = torch.randn(B, V, generator=g, device=cuda_device).to(dtype)
    history = torch.randint(0, V, (B, 200), generator=g, device=cuda_device)
    allowed = torch.rand(V, generator=g, device=cuda_device) < 0.7
    got = process_logits(x, history, repetition=1.3, frequency=0.5, allowed=allowed)
    for b in (0, 1, B // 2, B - 1):
        want = process_logits(x[b:b + 1], history[b:b + 1], repetition=1.3, frequency=0.5, allowed=allowed)
        assert torch.equal(got[b:b + 1], want)


def test_repetition_over_one_history_and_the_rest_over_another(cuda_device):
    """Two calls in float32 are one definition: with one history for both they are a single call, bit for bit."""
    from sparseforge_amd.logits import process_logits

    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(3, 1003, generator=g, device=cuda_device)
    history = torch.randint(0, 1003, (3, 400), generator=g, device=cuda_device)
    bias = torch.randn(1003, generator=g, device=cuda_device)
    allowed = torch.rand(1003, generator=g, device=cuda_device) < 0.8
    rest = dict(presence=0.7, frequency=0.3, bias=bias, allowed=allowed)
    once = process_logits(x, history, repetition=1.4, **rest)
    assert torch.equal(process_logits(process_logits(x, history, repetition=1.4), history, **rest), once)
    # the answer is the last 100 tokens
    got = process_logits(process_logits(x, history, repetition=1.4), history[:, 300:], **rest)
    count = torch.zeros(3, 1003, device=cuda_device).scatter_add_(1, history[:, 300:], torch.ones(3, 100, device=cuda_device))
    met = torch.zeros(3, 1003, dtype=torch.bool, device=cuda_device).scatter_(1, history, True)
    y = torch.where(met, torch.where(x > 0, x.double() / 1.4, x.double() * 1.4), x.double())
    y = y - torch.where(count > 0, 0.3 * count.double() + 0.7, 0.0) + bias
    assert bool(((got.double() - y).abs()[:, allowed] <= 1e-6 * (y.abs() + 10.0)[:, allowed]).all())
    assert bool((got[:, ~allowed] == -float("inf")).all())
