"""Cases of the training operators' edges that hold for the host twins and the
GPU alike (`where`: a device and the `stream` argument)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import mlx_cluster_amd as mc


def check_dual_tensors(where, grad_mode, requires_grad):
    """There is no forward-mode derivative: a call that would drop a tangent raises."""
    w = torch.randn(6, 4, device=where.device, requires_grad=requires_grad)
    plain = torch.randn(6, 4, device=where.device)
    x = torch.tensor([[0, 5, 2]], device=where.device)
    kw = dict(stream=where.stream)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = forward_ad.make_dual(w, torch.ones_like(plain))
        for call in (lambda: mc.embedding(dual, x, **kw), lambda: mc.window_scores(dual, x, 2, **kw),
                     lambda: mc.preference_loss(dual, plain, **kw),
                     lambda: mc.preference_loss(plain, dual, **kw)):
            with pytest.raises(NotImplementedError):
                call()
        mc.embedding(plain, x, **kw)  # others go on as they did
    mc.embedding(w.detach(), x, **kw)
