"""Cases of the training operators that hold for the host twins and the GPU
alike: each function takes the `stream` argument and a device, and checks one
operator against tests/train_reference.py."""
import itertools

import pytest
import torch

import mlx_cluster_amd as mc
import train_reference as ref

FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def table(g, V, D, dtype, layout="plain"):
    """[V, D]: in one piece, columns of a wider table (rows apart, and not on
    a 16-byte boundary), or rows that are transposed columns."""
    if layout == "wide":
        return torch.randn(V, D + 5, generator=g).to(dtype)[:, 3:3 + D]
    if layout == "turned":
        return torch.randn(D, V, generator=g).to(dtype).t()
    return torch.randn(V, D, generator=g).to(dtype)


def check_embedding(where, dtype, D, V, shape, int32, missing, scale, layout):
    g = gen(D, V, int32)
    w = table(g, V, D, dtype, layout)
    x = ref.make_nodes(g, shape, V, missing)
    if int32:
        x = x.int()
    got = mc.embedding(w.to(where.device), x.to(where.device), scale=scale, stream=where.stream)
    assert got.dtype == dtype and got.shape == (*shape, D)
    ref.close(got, *ref.embedding(w, x, scale))


EMBEDDING = [(dt, D, V, shape, i32, miss, s, lay) for (dt, D, (V, shape), (i32, miss, s), lay) in [
    (torch.float32, 64, (2708, (50,)), (False, 0.0, 1.0), "plain"),
    (torch.bfloat16, 128, (1000, (3, 41)), (True, 0.1, 11.3), "plain"),
    (torch.float16, 100, (77, (9, 2, 5)), (False, 0.5, 0.1), "plain"),
    (torch.float32, 1, (1, (1,)), (True, 0.0, -2.0), "plain"),
    (torch.bfloat16, 7, (5, (300,)), (False, 0.9, 1.0), "wide"),
    (torch.float16, 33, (64, (65,)), (True, 0.0, 3.0), "wide"),
    (torch.float32, 260, (10, (4, 4)), (False, 1.0, 1.0), "wide"),
    (torch.bfloat16, 16, (31, (127,)), (False, 0.2, 1.0), "turned"),
    (torch.bfloat16, 64, (9, (0,)), (False, 0.0, 1.0), "plain"),
    (torch.float32, 8, (0, (5,)), (False, 1.0, 1.0), "plain"),
    (torch.float16, 1030, (6, (3,)), (False, 0.0, 1.0), "plain"),
]]


def check_embedding_grad(where, dtype, out_dtype, D, V, count, int32, missing, hub, scale, sparse):
    g = gen(D, V, count, sparse)
    x = ref.make_nodes(g, (count,), V, missing, hub)
    if int32:
        x = x.int()
    gr = torch.randn(count, D, generator=g).to(dtype)
    got = mc.embedding_grad(gr.to(where.device), x.to(where.device), V, scale=scale, sparse=sparse,
                            out_dtype=out_dtype, stream=where.stream)
    want = ref.embedding_grad(gr, x, V, scale, out_dtype or dtype, sparse)
    if sparse:
        assert got[0].dtype == torch.int64 and torch.equal(got[0].cpu(), want[0])
        got, want = got[1], want[1:]
    assert got.dtype == (out_dtype or dtype)
    ref.close(got, *want)


EMBEDDING_GRAD = [(dt, od, D, V, T, i32, miss, hub, s, sparse) for (dt, od, D, V, T, i32, miss, hub, s), sparse in
                  itertools.product([
    (torch.float32, None, 64, 300, 1000, False, 0.0, 0.0, 1.0),
    (torch.float32, None, 1, 1, 1, False, 0.0, 0.0, 2.0),
    (torch.bfloat16, None, 128, 50, 700, True, 0.1, 0.6, 11.3),
    (torch.bfloat16, torch.float32, 100, 1000, 500, False, 0.5, 0.0, 0.1),
    (torch.float16, None, 33, 7, 321, False, 0.0, 0.9, 1.0),
    (torch.float32, torch.bfloat16, 7, 100, 64, True, 0.0, 1.0, 1.0),   # one full tile of one node
    (torch.float32, torch.float16, 16, 3, 4161, False, 0.0, 0.95, 1.0),  # tiles of tiles
    (torch.float16, None, 260, 5, 130, False, 1.0, 0.0, 1.0),            # no node at all
    (torch.float32, None, 8, 70000, 200, False, 0.0, 0.0, 1.0),          # three digits
    (torch.float32, None, 4, 256, 300, False, 0.0, 0.0, 1.0),            # exactly one digit
    (torch.float32, None, 4, 257, 300, False, 0.0, 0.0, 1.0),
    (torch.float32, None, 5, 10, 0, False, 0.0, 0.0, 1.0),
    (torch.float32, None, 5, 0, 12, False, 1.0, 0.0, 1.0),
    (torch.bfloat16, None, 1030, 4, 70, False, 0.0, 0.0, 1.0),
], [False, True])]


def check_window_scores(where, dtype, D, V, walks, int32, missing, scale, layout):
    N, M, C = walks
    g = gen(D, V, N, M, C)
    w = table(g, V, D, dtype, layout)
    x = ref.make_nodes(g, (N, M), V, missing)
    if int32:
        x = x.int()
    got = mc.window_scores(w.to(where.device), x.to(where.device), C, scale=scale,
                           stream=where.stream)
    assert got.dtype == torch.float32
    ref.close(got, *ref.window_scores(w, x, C, scale))
    windows = mc.context_windows(x.to(where.device), C, stream=where.stream)
    as_windows = mc.window_scores(w.to(where.device), windows, scale=scale, stream=where.stream)
    want, bound = ref.window_scores(w, windows.cpu(), C, scale)
    ref.close(as_windows, want, bound)


def check_window_scores_grad(where, dtype, out_dtype, D, V, walks, int32, missing, scale, sparse,
                             layout):
    N, M, C = walks
    g = gen(D, V, N, M, C)
    w = table(g, V, D, dtype, layout)
    x = ref.make_nodes(g, (N, M), V, missing, hub=0.1)
    if int32:
        x = x.int()
    gr = torch.randn(N, M - C + 1, C - 1, generator=g)
    want = ref.window_scores_grad(gr, w, x, C, scale, out_dtype or dtype, sparse)
    # pairs with no node: whatever the gradient holds there
    valid = x >= 0
    for k in range(1, C):
        both = valid[:, :M - C + 1] & valid[:, k:k + M - C + 1]
        gr[:, :, k - 1][~both] = float("nan")
    got = mc.window_scores_grad(gr.to(where.device), w.to(where.device), x.to(where.device), C,
                                scale=scale, sparse=sparse, out_dtype=out_dtype,
                                stream=where.stream)
    if sparse:
        assert torch.equal(got[0].cpu(), want[0])
        got, want = got[1], want[1:]
    assert got.dtype == (out_dtype or dtype)
    ref.close(got, *want)


WINDOW_SCORES = []
for _i, (_walks, _D) in enumerate(itertools.product(ref.WINDOWS, [1, 16, 33, 100, 128, 260])):
    WINDOW_SCORES.append((FLOATS[_i % 3], _D, [40, 3, 1000][_i // 2 % 3], _walks, _i % 2 == 1,
                          [0.0, 0.3][_i // 3 % 2], [1.0, 0.37][_i % 2],
                          ["plain", "wide"][_i // 5 % 2]))
WINDOW_SCORES += [(dt, D, 50, (3, 20, 6), False, 0.1, 1.0, "plain") for dt in FLOATS
                  for D in ref.DIMS]
WINDOW_SCORES += [(torch.float32, 32, 10, (0, 12, 4), False, 0.0, 1.0, "plain"),
                  (torch.bfloat16, 64, 10, (4, 12, 4), False, 1.0, 1.0, "plain")]


def check_preference(where, dtype, B, Tc, Tr, refs, masks, beta, smoothing, normalize, reduction,
                     masked_value=0.0):
    g = gen(B, Tc, Tr)
    sides = []
    for T in (Tc, Tr):
        v = torch.randn(B, T, generator=g)
        r = torch.randn(B, T, generator=g).to(dtype) if refs else None
        m = None
        if masks:
            m = torch.rand(B, T, generator=g) < torch.rand(B, 1, generator=g)
            m[::5] = False  # nothing left
            v[~m] = masked_value
            if refs:
                r[~m] = masked_value
        sides.append((v.to(dtype), r, m))
    to = lambda t: None if t is None else t.to(where.device)
    (c, rc, mcm), (r, rr, mrm) = [[to(t) for t in s] for s in sides]
    kw = dict(chosen_mask=mcm, rejected_mask=mrm, beta=beta, label_smoothing=smoothing,
              normalize=normalize, reduction=reduction, stream=where.stream)
    want = ref.preference(sides, beta, smoothing, normalize, reduction == "sum")
    got = mc.preference_loss_grad(c, r, rc, rr, **kw)
    for x, (value, bound) in zip(got, want):
        ref.close(x, value, bound)
    assert got[2].dtype == dtype and got[3].dtype == dtype
    loss, rewards = mc.preference_loss(c, r, rc, rr, return_rewards=True, **kw)
    assert torch.equal(loss, got[0]) and torch.equal(rewards, got[1])
    # through autograd, with a factor of its own
    c2, r2 = c.clone().requires_grad_(), r.clone().requires_grad_()
    loss = mc.preference_loss(c2, r2, rc, rr, **kw)
    (loss * 3.0).backward()
    for x, (value, bound) in zip((c2.grad, r2.grad), want[2:]):
        ref.close(x, 3 * value, 3 * bound * 1.01 + 3 * 2.0**-24 * value.abs())


PREFERENCE = [
    (torch.float32, 1, 1, 1, False, False, 0.1, 0.0, False, "mean"),
    (torch.float32, 2000, 5, 5, False, False, 1.0, 0.0, False, "mean"),
    (torch.float32, 333, 9, 9, True, False, 0.5, 0.1, False, "sum"),
    (torch.bfloat16, 65, 31, 77, True, True, 0.1, 0.1, True, "sum"),
    (torch.float16, 17, 130, 64, True, True, 2.0, 0.0, False, "sum"),
    (torch.float32, 3, 2049, 5, False, True, 0.3, 1.0, True, "mean"),
    (torch.bfloat16, 4, 1025, 777, True, True, 0.1, 0.5, True, "mean"),
    (torch.float32, 129, 16, 17, True, True, -0.4, 0.2, False, "mean"),
    (torch.float32, 40, 3, 0, False, False, 1.0, 0.0, False, "mean"),
    (torch.float32, 40, 0, 0, False, False, 1.0, 0.0, True, "sum"),
    (torch.float16, 0, 4, 6, False, False, 1.0, 0.0, False, "mean"),
    (torch.bfloat16, 1001, 9, 33, False, True, 0.7, 0.0, True, "sum"),
    (torch.float32, 7, 64, 257, True, True, 0.0, 0.0, False, "mean"),
    (torch.float32, 2, 5000, 4999, True, True, 0.05, 0.0, False, "mean"),
]
MASKED_VALUES = [0.0, float("-inf"), float("inf"), float("nan"), "lowest"]


def lowest(dtype):
    return torch.finfo(dtype).min
