"""The training operators' host twins, arguments and C ABI (CPU only)."""
import ctypes
import os
import re
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import mlx_cluster_amd as mc
import train_cases as cases
import train_reference as ref
from mlx_cluster_amd import _lib

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "mlxc_train.h")
CPU = SimpleNamespace(device=torch.device("cpu"), stream="cpu")


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(mlxc_\w+)\s*\(", text)))
    assert declared == sorted(_lib.TRAIN_SIGNATURES)
    lib = _lib.load()
    assert all(hasattr(lib, name) for name in declared)
    for name in ["MLXC_FLOAT32", "MLXC_BFLOAT16", "MLXC_FLOAT16", "MLXC_GRAD_SPARSE",
                 "MLXC_PREFERENCE_NORMALIZE", "MLXC_PREFERENCE_SUM"]:
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == getattr(_lib, name)


@pytest.mark.parametrize("case", cases.EMBEDDING)
def test_embedding(case):
    cases.check_embedding(CPU, *case)


@pytest.mark.parametrize("case", cases.EMBEDDING_GRAD)
def test_embedding_grad(case):
    cases.check_embedding_grad(CPU, *case)


@pytest.mark.parametrize("case", cases.WINDOW_SCORES[::4])
def test_window_scores(case):
    cases.check_window_scores(CPU, *case)


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("case", cases.WINDOW_SCORES[1::6])
def test_window_scores_grad(case, sparse):
    dtype, D, V, walks, int32, missing, scale, layout = case
    cases.check_window_scores_grad(CPU, dtype, None, D, V, walks, int32, missing, scale, sparse,
                                   layout)


@pytest.mark.parametrize("case", cases.PREFERENCE)
def test_preference(case):
    cases.check_preference(CPU, *case)


@pytest.mark.parametrize("value", cases.MASKED_VALUES)
def test_preference_masked_values(value):
    for dtype in cases.FLOATS:
        v = cases.lowest(dtype) if value == "lowest" else value
        cases.check_preference(CPU, dtype, 33, 11, 20, True, True, 0.5, 0.1, True, "sum", v)


def test_infinite_ratios():
    # a probability of 0 on one side: the loss is infinite or 0, its slope finite
    inf = float("inf")
    c = torch.tensor([[-inf, 0.0], [0.0, 0.0], [-inf, 0.0]])
    r = torch.tensor([[0.0, 0.0], [-inf, 0.0], [0.0, -1.0]])
    loss, rewards, dc, dr = mc.preference_loss_grad(c[1:2], r[1:2], beta=1.0, stream="cpu")
    assert float(loss) == 0 and torch.equal(dc, torch.zeros(1, 2)) and torch.equal(dr, -dc)
    loss, rewards, dc, dr = mc.preference_loss_grad(c[:1], r[:1], beta=1.0, stream="cpu")
    assert float(loss) == inf and torch.equal(dc, -torch.ones(1, 2)) and torch.equal(dr, -dc)


# ---- gradients against differences, in 64 bits on the formulas and here


def test_gradients_against_differences():
    g = cases.gen(1)
    V, D, C = 12, 6, 4
    w = torch.randn(V, D, generator=g)
    walks = ref.make_nodes(g, (5, 9), V, 0.1, 0.2)
    neg = ref.make_nodes(g, (30, C), V, 0.0)

    def loss64(w64):
        pos = ref.window_scores(w64, walks, C, 0.5)[0].reshape(30, C - 1)
        other = ref.window_scores(w64, neg, C, 0.5)[0].reshape(30, C - 1)
        rows = ref.rows_of(w64, walks)[0] * 2.0
        z = 0.7 * (pos.sum(-1) - other.sum(-1))
        return torch.nn.functional.softplus(-z).mean() + 0.01 * (rows**2).sum()

    p = w.clone().requires_grad_()
    pos = mc.window_scores(p, walks, C, scale=0.5, stream="cpu")
    other = mc.window_scores(p, neg, scale=0.5, stream="cpu").reshape(pos.shape)
    loss = mc.preference_loss(pos.reshape(30, -1), other.reshape(30, -1), beta=0.7, stream="cpu")
    rows = mc.embedding(p, walks, scale=2.0, stream="cpu")
    (loss + 0.01 * (rows**2).sum()).backward()
    h = 1e-5
    for v in range(V):
        for d in range(D):
            a, b = w.double().clone(), w.double().clone()
            a[v, d] += h
            b[v, d] -= h
            slope = (loss64(a) - loss64(b)) / (2 * h)
            # a difference's own error is h^2 of the third derivative and
            # 1e-16 / h of the values; float32 sums give the rest
            assert abs(float(slope) - float(p.grad[v, d])) < 1e-5 * (1 + abs(float(slope)))


def test_sparse_autograd_gradient():
    g = cases.gen(2)
    w = torch.randn(20, 5, generator=g)
    x = ref.make_nodes(g, (4, 7), 20, 0.3)
    grads = []
    for sparse in (False, True):
        p = w.clone().requires_grad_()
        (mc.embedding(p, x, scale=3.0, sparse_grad=sparse, stream="cpu") ** 2).sum().backward()
        s = mc.window_scores(p, x, 3, sparse_grad=sparse, stream="cpu")
        q = w.clone().requires_grad_()
        mc.window_scores(q, x, 3, sparse_grad=sparse, stream="cpu").sum().backward()
        assert s.requires_grad and q.grad.is_sparse == sparse and p.grad.is_sparse == sparse
        grads.append((p.grad.to_dense(), q.grad.to_dense()))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


# ---- refusals


def test_refusals():
    w, x = torch.randn(4, 3), torch.tensor([[0, 1, 2]])
    s = mc.window_scores(w, x, 2, stream="cpu")
    bad = [
        (TypeError, lambda: mc.embedding(w.double(), x, stream="cpu")),
        (TypeError, lambda: mc.embedding("w", x, stream="cpu")),
        (ValueError, lambda: mc.embedding(w[0], x, stream="cpu")),
        (ValueError, lambda: mc.embedding(w[:, :0], x, stream="cpu")),
        (TypeError, lambda: mc.embedding(w, x.float(), stream="cpu")),
        (TypeError, lambda: mc.embedding(w, x, scale="1", stream="cpu")),
        (TypeError, lambda: mc.embedding(w, x, stream=3)),
        (ValueError, lambda: mc.embedding(w, x + 2, stream="cpu")),
        (ValueError, lambda: mc.embedding(w, x - 2, stream="cpu")),
        (ValueError, lambda: mc.embedding_grad(w, x, 4, stream="cpu")),
        (ValueError, lambda: mc.embedding_grad(torch.randn(1, 3, 2), x, -1, stream="cpu")),
        (TypeError, lambda: mc.embedding_grad(torch.randn(1, 3, 2), x, 4.0, stream="cpu")),
        (TypeError, lambda: mc.embedding_grad(torch.randn(1, 3, 2), x, 4, out_dtype=torch.int32,
                                              stream="cpu")),
        (ValueError, lambda: mc.embedding_grad(torch.randn(1, 3, 2), x, 2, stream="cpu")),
        (ValueError, lambda: mc.window_scores(w, x[0], 2, stream="cpu")),
        (ValueError, lambda: mc.window_scores(w, x, 1, stream="cpu")),
        (ValueError, lambda: mc.window_scores(w, x, 4, stream="cpu")),
        (ValueError, lambda: mc.window_scores(w, torch.zeros(1, 40).long(), stream="cpu")),
        (TypeError, lambda: mc.window_scores(w, x, 2.0, stream="cpu")),
        (ValueError, lambda: mc.window_scores_grad(s[:, :1], w, x, 2, stream="cpu")),
        (TypeError, lambda: mc.window_scores_grad(s.half(), w, x, 2, stream="cpu")),
        (ValueError, lambda: mc.window_scores_grad(s, w, x + 5, 2, stream="cpu")),
        (ValueError, lambda: mc.preference_loss(w, w[:3], stream="cpu")),
        (TypeError, lambda: mc.preference_loss(w, w.half(), stream="cpu")),
        (TypeError, lambda: mc.preference_loss(w, w, w.half(), stream="cpu")),
        (ValueError, lambda: mc.preference_loss(w, w, w[:, :2], stream="cpu")),
        (ValueError, lambda: mc.preference_loss(w, w, chosen_mask=w[:, :2] > 0, stream="cpu")),
        (TypeError, lambda: mc.preference_loss(w, w, chosen_mask=w, stream="cpu")),
        (ValueError, lambda: mc.preference_loss(w, w, beta=float("inf"), stream="cpu")),
        (ValueError, lambda: mc.preference_loss(w, w, label_smoothing=1.5, stream="cpu")),
        (ValueError, lambda: mc.preference_loss(w, w, reduction="none", stream="cpu")),
        (ValueError, lambda: mc.preference_loss(torch.tensor(1.0), w, stream="cpu")),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()


def test_unchecked_bad_nodes_are_no_nodes():
    g = cases.gen(3)
    w = torch.randn(5, 4, generator=g)
    x = torch.tensor([[0, 7, 2, -3, 4, 2**40]])
    y = torch.where((x >= 0) & (x < 5), x, -1)
    kw = dict(check=False, stream="cpu")
    assert torch.equal(mc.embedding(w, x, **kw), mc.embedding(w, y, **kw))
    s = mc.window_scores(w, x, 3, **kw)
    assert torch.equal(s, mc.window_scores(w, y, 3, **kw))
    gr = torch.randn(s.shape, generator=g)
    assert torch.equal(mc.window_scores_grad(gr, w, x, 3, **kw),
                       mc.window_scores_grad(gr, w, y, 3, **kw))


FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: the checks fail first
SIDE = _lib.PreferenceSide(0x1000, None, None, 4, None)


@pytest.mark.parametrize("name,args,msg", [
    ("mlxc_embedding", (FAKE, -1, 4, 4, 0, FAKE, 1, 0, 1.0, FAKE, None, None), "num_rows"),
    ("mlxc_embedding", (FAKE, 2**31, 4, 4, 0, FAKE, 1, 0, 1.0, FAKE, None, None), "num_rows"),
    ("mlxc_embedding", (FAKE, 1, 0, 4, 0, FAKE, 1, 0, 1.0, FAKE, None, None), "dim"),
    ("mlxc_embedding", (FAKE, 1, 4, 3, 0, FAKE, 1, 0, 1.0, FAKE, None, None), "row_stride"),
    ("mlxc_embedding", (FAKE, 1, 4, 4, 3, FAKE, 1, 0, 1.0, FAKE, None, None), "dtype"),
    ("mlxc_embedding", (FAKE, 1, 4, 4, 0, FAKE, -1, 0, 1.0, FAKE, None, None), ">= 0"),
    ("mlxc_embedding", (FAKE, 1, 4, 4, 0, FAKE, 1, 2, 1.0, FAKE, None, None), "node_type"),
    ("mlxc_embedding", (None, 1, 4, 4, 0, FAKE, 1, 0, 1.0, FAKE, None, None), "weight"),
    ("mlxc_embedding", (FAKE, 1, 4, 4, 0, None, 1, 0, 1.0, FAKE, None, None), "nodes"),
    ("mlxc_embedding", (FAKE, 1, 4, 4, 0, FAKE, 1, 0, 1.0, ctypes.c_void_p(0x1002), None, None),
     "aligned"),
    ("mlxc_embedding_grad", (FAKE, 4, 0, FAKE, 2**31 - 1, 0, 9, 1.0, 0, None, FAKE, 0, FAKE, 1 << 40,
                             None), "split"),
    ("mlxc_embedding_grad", (FAKE, 4, 0, FAKE, 5, 0, 9, 1.0, 1, None, FAKE, 0, FAKE, 1 << 40, None),
     "ids"),
    ("mlxc_embedding_grad", (FAKE, 4, 0, FAKE, 5, 0, 9, 1.0, 2, None, FAKE, 0, FAKE, 1 << 40, None),
     "flags"),
    ("mlxc_embedding_grad", (FAKE, 4, 0, FAKE, 5, 0, 9, 1.0, 0, None, FAKE, 9, FAKE, 1 << 40, None),
     "out_dtype"),
    ("mlxc_embedding_grad", (FAKE, 4, 0, FAKE, 5, 0, 9, 1.0, 0, None, FAKE, 0, FAKE, 100, None),
     "workspace holds"),
    ("mlxc_embedding_grad", (FAKE, 4, 0, FAKE, 5, 0, 9, 1.0, 0, None, FAKE, 0,
                             ctypes.c_void_p(0x1008), 1 << 40, None), "16-byte"),
    ("mlxc_window_scores", (FAKE, 9, 4, 4, 0, FAKE, 1, 8, 1, 0, 1.0, FAKE, None, None), "context"),
    ("mlxc_window_scores", (FAKE, 9, 4, 4, 0, FAKE, 1, 80, 33, 0, 1.0, FAKE, None, None), "context"),
    ("mlxc_window_scores", (FAKE, 9, 4, 4, 0, FAKE, 2**28, 8, 3, 0, 1.0, FAKE, None, None), "split"),
    ("mlxc_window_scores", (FAKE, 9, 4, 4, 0, FAKE, 2**62, 8, 3, 0, 1.0, FAKE, None, None), "split"),
    ("mlxc_window_scores", (FAKE, 9, 4, 4, 0, FAKE, 1, 8, 3, 0, 1.0, None, None, None), "scores"),
    ("mlxc_window_scores_grad", (None, FAKE, 9, 4, 4, 0, FAKE, 1, 8, 3, 0, 1.0, 0, None, FAKE, 0,
                                 FAKE, 1 << 40, None), "grad"),
    ("mlxc_preference_loss", (SIDE, SIDE, -1, 0, 1.0, 0.0, 0, FAKE, None, None, FAKE, 1 << 30, None),
     "pairs"),
    ("mlxc_preference_loss", (SIDE, SIDE, 2, 5, 1.0, 0.0, 0, FAKE, None, None, FAKE, 1 << 30, None),
     "dtype"),
    ("mlxc_preference_loss", (SIDE, SIDE, 2, 0, 1.0, 0.0, 4, FAKE, None, None, FAKE, 1 << 30, None),
     "flags"),
    ("mlxc_preference_loss", (SIDE, SIDE, 2, 0, 1.0, 0.0, 0, None, None, None, FAKE, 1 << 30, None),
     "loss"),
    ("mlxc_preference_loss", (SIDE, SIDE, 2, 0, 1.0, 0.0, 0, FAKE, None, None, FAKE, 0, None),
     "workspace holds"),
    ("mlxc_preference_loss", (None, SIDE, 2, 0, 1.0, 0.0, 0, FAKE, None, None, FAKE, 64, None),
     "NULL"),
    ("mlxc_preference_grad", (SIDE, SIDE, 2, 0, None, None, None), "slopes"),
])
def test_c_entries_refuse(name, args, msg):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == _lib.MLXC_ERR_INVALID_ARGUMENT
    assert msg in _lib.last_error()


def test_workspace_queries():
    lib = _lib.load()
    assert lib.mlxc_embedding_grad_workspace_bytes(10, 4, -1, 0) == 0
    assert lib.mlxc_embedding_grad_workspace_bytes(10, 4, 2**31 - 1, 0) == 0
    assert lib.mlxc_embedding_grad_workspace_bytes(10, 4, 0, 0) > 0
    assert lib.mlxc_window_scores_grad_workspace_bytes(10, 4, 3, 8, 9, 0) == 0
    assert (lib.mlxc_window_scores_grad_workspace_bytes(10, 4, 3, 8, 4, 0) >=
            lib.mlxc_embedding_grad_workspace_bytes(10, 4, 24, 0) + 24 * 4 * 4)


def test_numpy_arguments():
    w = np.random.default_rng(0).standard_normal((6, 4)).astype(np.float32)
    x = np.array([0, 5, -1])
    got = mc.embedding(w, x, stream="cpu")
    assert np.array_equal(got.numpy()[:2], w[[0, 5]]) and not got.numpy()[2].any()


def test_half_conversions_of_the_host_twins():
    # every float16 and bfloat16 comes back as itself; halves of steps go to even
    for dtype in (torch.float16, torch.bfloat16):
        w = torch.arange(-2**15, 2**15).to(torch.int16).view(dtype).reshape(-1, 1)
        got = mc.embedding(w, torch.arange(2**16), stream="cpu")
        nan = torch.isnan(w)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan].view(torch.int16), w[~nan].view(torch.int16))
        f = torch.randn(4000, 1, generator=cases.gen(5)) * 10.0**torch.linspace(-42, 39, 4000)[:, None]
        got = mc.embedding_grad(f, torch.arange(4000), 4000, out_dtype=dtype, stream="cpu")
        assert torch.equal(got, f.to(dtype))


def test_example_trains_on_the_cpu():
    """examples/train_embeddings.py: the operators together, on their host twins."""
    from conftest import REPO
    import importlib.util
    spec = importlib.util.spec_from_file_location(
        "train_embeddings", os.path.join(REPO, "examples", "train_embeddings.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first, last, right = example.train(nodes=1000, steps=40, batch=500, labelled=0.05, device="cpu",
                                       log=lambda *a: None)
    # losses start at log 2 (no preference); classes by chance are right in one of five
    assert abs(first[0] - 0.6931) < 0.02 and max(last) < 0.6 and right > 0.6
