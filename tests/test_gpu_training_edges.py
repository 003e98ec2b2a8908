"""The training operators' kernels at row sizes, table sizes and ways to call
that lie between those of test_gpu_training.py."""
from types import SimpleNamespace

import pytest
import torch

import mlx_cluster_amd as mc
import train_cases as cases
import train_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return SimpleNamespace(device=torch.device("cuda", 0), stream=None)


# Row sizes that are whole steps of a matrix instruction (16 float32, 32 16-bit
# values) but fewer of them than the kernel holds (1, 2, 4, 8, or 4 at a time).
STEPS = [(torch.float32, D) for D in (48, 80, 96, 112, 144, 176, 208, 240, 272)] + \
    [(dt, D) for dt in (torch.bfloat16, torch.float16) for D in (96, 160, 192, 224, 288, 320, 352)]


@pytest.mark.parametrize("walks", [(3, 40, 17), (7, 81, 10), (4, 33, 32), (5, 9, 9)])
@pytest.mark.parametrize("dtype,D", STEPS)
def test_scores_of_rows_of_whole_steps(gpu, dtype, D, walks):
    cases.check_window_scores(gpu, dtype, D, 50, walks, False, 0.1, 0.7, "plain")
    cases.check_window_scores_grad(gpu, dtype, None, D, 50, walks, True, 0.1, 0.7, False, "plain")
