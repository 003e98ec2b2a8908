"""The training operators' host twins and arguments where test_training.py's
cases do not reach (CPU only)."""
from types import SimpleNamespace

import pytest
import torch

import train_edges as edges

CPU = SimpleNamespace(device=torch.device("cpu"), stream="cpu")


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_dual_tensors_are_refused(grad_mode, requires_grad):
    edges.check_dual_tensors(CPU, grad_mode, requires_grad)


def test_sizes_past_32_bits():
    edges.check_sizes_past_32_bits(CPU)
