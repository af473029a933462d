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
