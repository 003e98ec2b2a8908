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


def check_sizes_past_32_bits(where):
    """Sizes that a 32-bit number would cut are refused by what they are."""
    kw = dict(stream=where.stream)
    d = where.device
    none, x = torch.zeros(0, dtype=torch.int64, device=d), torch.zeros(2, 3, dtype=torch.int64, device=d)
    w = torch.zeros(4, 8, device=d)
    for D in (65537, 2**31, 2**32 + 4):
        wide = torch.empty(0, D, dtype=torch.float16, device=d)  # no memory
        for call in (lambda: mc.embedding(wide, none, **kw),
                     lambda: mc.embedding(wide.clone().requires_grad_(), none, **kw),
                     lambda: mc.window_scores(wide, x - 1, 2, **kw),
                     lambda: mc.window_scores_grad(torch.zeros(2, 2, 1, device=d), wide, x - 1, 2, **kw),
                     lambda: mc.embedding_grad(wide, none, 0, **kw),
                     lambda: mc.embedding_grad(wide, none, 0, sparse=True, out_dtype=torch.float32,
                                               **kw)):
            with pytest.raises(ValueError, match="dim"):
                call()
    for M in (2**31, 2**32 + 5):
        long = torch.empty(0, M, dtype=torch.int64, device=d)
        with pytest.raises(ValueError, match="walks of at most"):
            mc.window_scores(w, long, 4, **kw)
        with pytest.raises(ValueError, match="walks of at most"):
            mc.window_scores_grad(torch.empty(0, M - 3, 3, device=d), w, long, 4, **kw)
    g = torch.zeros(2, 3, 8, device=d)
    for V in (2**31, 2**32 + 5, 2**64 + 5):
        for sparse in (False, True):
            with pytest.raises(ValueError, match="num_nodes"):
                mc.embedding_grad(g, x, V, sparse=sparse, **kw)
    for C in (2**31 + 2, 2**32 + 2, 2**64 + 2):
        with pytest.raises(ValueError, match="context_size"):
            mc.window_scores(w, x, C, **kw)
