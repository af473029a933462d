"""Distillation from a teacher's top logits through Distill_Model and RetrainStep: the teacher recorded, or run."""
import itertools

import pytest
import torch
from test_gpu_retrain import _build

pytestmark = pytest.mark.gpu


def _batches(dev, n=2):
    g = torch.Generator(device=dev).manual_seed(11)
    return [tuple(torch.randint(0, 512, (2, 24), generator=g, device=dev) for _ in range(2)) for _ in range(n)]


def _record(teacher, batches, k):
    from sparseforge_amd.distill import top_logits

    with torch.no_grad():
        return [(X, Y, top_logits(teacher(X, Y)[0], k)) for X, Y in batches]


def test_distill_model_from_the_top(cuda_device):
    """The teacher's top logits taken on the way, and a record of them, give the loss and gradients of top_kl_loss."""
    from sparseforge_amd.distill import top_kl_loss, top_logits
    from sparseforge_amd.sparse_modeling import Distill_Model

    _, student, teacher, _, _ = _build(cuda_device)
    (X, Y), = _batches(cuda_device, 1)
    params = [p for p in student.parameters() if p.requires_grad]

    def grads(loss):
        return torch.autograd.grad(loss, params, allow_unused=True)

    logits, task, layerwise, kl = Distill_Model(student, teacher, top=32)(X, Y)
    assert layerwise is None
    with torch.no_grad():
        top = top_logits(teacher(X, Y)[0], 32)
    want = top_kl_loss(student(X, Y)[0], top)
    assert float(kl.detach()) == float(want.detach())
    recorded = Distill_Model(student, None)(X, Y, top)
    assert float(recorded[3].detach()) == float(want.detach()) and torch.equal(recorded[0], logits)
    some = 0
    for a, b, c in zip(grads(want), grads(kl), grads(recorded[3])):
        assert (a is None) == (b is None) == (c is None)
        if a is not None:
            some += 1
            assert torch.equal(a, b) and torch.equal(a, c)
    assert some > 4
    with pytest.raises(ValueError):
        Distill_Model(student, teacher, output_hidden_state=True)(X, Y, top)
    student.config.output_hidden_state = False


def test_step_with_all_logits_recorded_is_the_whole_teachers(cuda_device):
    """With every logit in the record the step's loss is that of the whole teacher: the same KL, up to the float32 sums of
    512 terms in each (2e-6 of it), and the same task loss and penalties."""
    from sparseforge_amd.retrain import RetrainStep

    losses = []
    for record in (False, True):
        _, student, teacher, opt, rc = _build(cuda_device)
        batches = _batches(cuda_device)
        if record:
            batches = _record(teacher, batches, 512)
        losses.append(RetrainStep(student, None if record else teacher, opt, rc)(1, batches).loss)
    assert abs(losses[0] - losses[1]) <= 4e-6 * abs(losses[0])


@pytest.mark.parametrize("hutchinson", [True, False])
def test_steps_with_a_record_equal_steps_with_its_teacher(cuda_device, hutchinson, monkeypatch):
    """Teacher run with teacher_top, and the same teacher recorded: the same steps bit for bit, probes included (the KL is
    differentiated twice there)."""
    from sparseforge_amd import utils as U
    from sparseforge_amd.retrain import RetrainStep

    seen = []
    for record in (False, True):
        monkeypatch.setattr(U, "_seed_counter", itertools.count(1))  # the probes' and samples' seeds
        _, student, teacher, opt, rc = _build(cuda_device)
        rc.teacher_top, rc.hutchinson = 24, hutchinson
        batches = _batches(cuda_device)
        if record:
            batches = _record(teacher, batches, 24)
        step = RetrainStep(student, None if record else teacher, opt, rc)
        out = [step(i, batches) for i in (1, 2)]
        assert not any(o.skipped for o in out) and all(o.loss == o.loss for o in out)
        seen.append([o.loss for o in out] + [p.detach().clone() for p in student.parameters()])
    for a, b in zip(*seen):
        assert torch.equal(torch.as_tensor(a), torch.as_tensor(b))
