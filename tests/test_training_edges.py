"""The training operators' host twins and arguments where test_training.py's
cases do not reach (CPU only)."""
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

import train_edges as edges
from mlx_cluster_amd import _lib
from conftest import REPO

CPU = SimpleNamespace(device=torch.device("cpu"), stream="cpu")


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_dual_tensors_are_refused(grad_mode, requires_grad):
    edges.check_dual_tensors(CPU, grad_mode, requires_grad)


def test_sizes_past_32_bits():
    edges.check_sizes_past_32_bits(CPU)


HUGE_LISTS = """
import ctypes
from mlx_cluster_amd import _lib
lib = _lib.load()
fake = ctypes.c_void_p(0x1000)  # never dereferenced: its copy does not fit first
for count in (2**59, 2**60, 2**61 - 1):
    assert lib.mlxc_embedding_grad_cpu(fake, 1, 0, fake, count, 0, 9, 1.0, 0, None, fake, 0, None) == -2
    assert "memory" in _lib.last_error()
side = _lib.PreferenceSide(0x1000, None, None, 1, 0x1000)
for pairs in (2**58, 2**60, 2**61 - 1):
    assert lib.mlxc_preference_loss_cpu(side, side, pairs, 0, 1.0, 0.0, 0, fake, None, None) == -2
print("ok")
"""


def test_host_lists_larger_than_memory_are_errors():
    """No exception leaves a C entry (it would end the process: a process of its own here)."""
    run = subprocess.run([sys.executable, "-c", HUGE_LISTS], cwd=REPO, capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stderr


def test_short_lists_need_no_workspace_of_the_table():
    """A dense gradient of up to 16,384 places works in LDS: its workspace is the status words,
    whatever the table and the rows; the next place brings the sort's and the sums'."""
    lib = _lib.load()
    q = lib.mlxc_embedding_grad_workspace_bytes
    for V in (1, 1 << 24, 2**31 - 1):
        for D in (1, 256, 65536):
            for T in (1, 10, 16384):
                assert 64 <= q(V, D, T, 0) <= 256
    assert q(1 << 24, 64, 16385, 0) > 8 << 24
    assert q(1 << 24, 64, 10, _lib.MLXC_GRAD_SPARSE) > 64 + 10 * (4 + 4 + 8)
    w = lib.mlxc_window_scores_grad_workspace_bytes
    assert 24 * 64 * 4 + 64 <= w(1 << 24, 64, 3, 8, 4, 0) <= 24 * 64 * 4 + 512
