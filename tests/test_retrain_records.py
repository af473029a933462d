"""Batches without a record of the teacher's logits where there is no teacher: refused before anything runs, since they would
train without the distillation that is asked for."""
import types

import pytest
import torch

from sparseforge_amd.retrain import RetrainConfig, RetrainStep
from sparseforge_amd.sparse_modeling import Distill_Model


class _Student(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.config = types.SimpleNamespace()
        self.ran = 0

    def forward(self, idx, targets):
        self.ran += 1
        return torch.zeros(*idx.shape, 8), torch.zeros(()), None


X = torch.zeros(1, 3, dtype=torch.int64)


def test_distill_model_asked_for_the_top_needs_a_teacher_or_a_record():
    student = _Student()
    model = Distill_Model(student, None, top=4)
    with pytest.raises(ValueError, match="record"):
        model(X, X)
    assert student.ran == 0
    # as in the reference without either
    assert float(Distill_Model(student, None)(X, X)[3]) == 0.0


@pytest.mark.parametrize("top", [0, 4])
def test_a_step_without_a_teacher_needs_a_record_in_every_batch(top):
    student = _Student()
    step = RetrainStep(student, None, None, RetrainConfig(grad_accum=2, teacher_top=top, autocast_dtype=None))
    record = object()  # not looked at: the step is refused first
    for batches in ([(X, X), (X, X)], [(X, X, record), (X, X)], [(X, X, record), (X, X, None)]):
        with pytest.raises(ValueError, match="record"):
            step(1, batches)
    assert student.ran == 0


@pytest.mark.gpu
def test_steps_without_the_kl_need_no_teacher(cuda_device):
    from test_gpu_retrain import _build

    _, student, _, opt, rc = _build(cuda_device)
    rc.hardness_kldiv, rc.teacher_top, rc.hutchinson = 0.0, 8, False
    g = torch.Generator(device=cuda_device).manual_seed(1)
    batches = [tuple(torch.randint(0, 512, (2, 24), generator=g, device=cuda_device) for _ in range(2)) for _ in range(2)]
    out = RetrainStep(student, None, opt, rc)(1, batches)
    assert not out.skipped and out.loss == out.loss
