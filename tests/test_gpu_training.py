"""The training operators' kernels against the formulas in 64 bits, and the
ways they are called: streams, strides, workspaces, repeated calls."""
from types import SimpleNamespace

import pytest
import torch

import mlx_cluster_amd as mc
import train_cases as cases
import train_reference as ref
from mlx_cluster_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return SimpleNamespace(device=torch.device("cuda", 0), stream=None)


@pytest.mark.parametrize("case", cases.EMBEDDING)
def test_embedding(gpu, case):
    cases.check_embedding(gpu, *case)


@pytest.mark.parametrize("case", cases.EMBEDDING_GRAD)
def test_embedding_grad(gpu, case):
    cases.check_embedding_grad(gpu, *case)


@pytest.mark.parametrize("case", cases.WINDOW_SCORES)
def test_window_scores(gpu, case):
    cases.check_window_scores(gpu, *case)


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("case", cases.WINDOW_SCORES)
def test_window_scores_grad(gpu, case, sparse):
    dtype, D, V, walks, int32, missing, scale, layout = case
    out = cases.FLOATS[D % 3] if D % 2 else None
    cases.check_window_scores_grad(gpu, dtype, out, D, V, walks, int32, missing, scale, sparse,
                                   layout)


@pytest.mark.parametrize("case", cases.PREFERENCE)
def test_preference(gpu, case):
    cases.check_preference(gpu, *case)


@pytest.mark.parametrize("value", cases.MASKED_VALUES)
def test_preference_masked_values(gpu, value):
    for dtype in cases.FLOATS:
        for shape in ((33, 11, 20), (9, 300, 70)):
            v = cases.lowest(dtype) if value == "lowest" else value
            cases.check_preference(gpu, dtype, *shape, True, True, 0.5, 0.1, True, "sum", v)


def test_infinite_ratios(gpu):
    inf = float("inf")
    t = lambda *rows: torch.tensor(rows, device=gpu.device)
    loss, _, dc, dr = mc.preference_loss_grad(t([0.0, 0.0]), t([-inf, 0.0]), beta=1.0)
    assert float(loss) == 0 and not dc.any() and not dr.any()
    loss, _, dc, dr = mc.preference_loss_grad(t([-inf, 0.0]), t([0.0, 0.0]), beta=1.0)
    assert float(loss) == inf and (dc == -1).all() and (dr == 1).all()


# ---- larger calls: against the same sums in 64 bits


def sum_by_node(rows, at, V):
    """Rows added up by node, on the CPU: a hub's row takes most of the adds,
    and 64-bit atomics on the GPU that meet on one row take minutes."""
    return torch.zeros(V, rows.shape[1], dtype=torch.float64).index_add_(0, at, rows)


@pytest.mark.parametrize("V,T,D,dtype,hub,missing,sparse", [
    (1 << 20, 300_001, 64, torch.float32, 0.3, 0.0, False),
    (1 << 20, 300_001, 40, torch.bfloat16, 0.0, 0.5, True),
    (100_003, 700_000, 17, torch.float16, 0.9, 0.1, False),
    (3, 600_000, 8, torch.float32, 0.5, 0.0, True),
    (1 << 24, 50_000, 4, torch.float32, 0.0, 0.0, True),
    (5000, 20_000, 128, torch.float32, 0.1, 0.1, False),
])
def test_embedding_grad_large(gpu, V, T, D, dtype, hub, missing, sparse):
    g = cases.gen(V, T, D)
    x = ref.make_nodes(g, (T,), V, missing, hub).to(gpu.device)
    gr = torch.randn(T, D, generator=g).to(dtype).to(gpu.device)
    got = mc.embedding_grad(gr, x, V, scale=0.5, sparse=sparse)
    keep = (x >= 0).cpu()
    at = x.cpu()[keep]
    n = torch.bincount(at, minlength=V).double()
    if sparse:
        ids = torch.nonzero(n).flatten()
        cap = min(V, T)
        assert torch.equal(got[0][:ids.numel()].cpu(), ids)
        assert (got[0][ids.numel():] == -1).all() and got[0].numel() == cap
        assert not got[1][ids.numel():].any()
        got = got[1][:ids.numel()]
    for lo in range(0, D, 16):  # columns at a time: 64-bit copies of the table
        cols = gr[:, lo:lo + 16].cpu()[keep].double()
        total, size = sum_by_node(cols, at, V), sum_by_node(cols.abs(), at, V)
        value, bound = ref.stored(total * 0.5, (n.unsqueeze(1) + 4) * ref.U32 * size * 0.5, dtype)
        if sparse:
            value, bound = value[ids], bound[ids]
        off = (got[:, lo:lo + 16].cpu().double() - value).abs() - bound
        assert float(off.max()) <= 0
    again = mc.embedding_grad(gr, x, V, scale=0.5, sparse=sparse)
    assert torch.equal(got, again[1][:got.shape[0]] if sparse else again)


@pytest.mark.parametrize("T", [1, 31, 32, 33, 1023, 1025, 4096, 16383, 16384, 16385, 20481, 65536, 65537,
                               262144, 262145, 300000])
@pytest.mark.parametrize("V", [1, 200, 256, 257, 65537, 1 << 20])
def test_sort_sizes(gpu, T, V):
    """Lists on both sides of every limit of the sort: exact sums of small whole numbers,
    nodes missing and bad, both forms, the status each time."""
    g = cases.gen(T, V)
    x = ref.make_nodes(g, (T,), V, 0.1, 0.2)
    gr = torch.randint(-8, 9, (T, 3), generator=g).float()
    keep = x >= 0
    want = torch.zeros(V, 3).index_add_(0, x[keep], gr[keep])
    ids = torch.unique(x[keep])
    out = mc.embedding_grad(gr.to(gpu.device), x.to(gpu.device), V)
    assert torch.equal(out.cpu(), want)
    got_ids, rows = mc.embedding_grad(gr.to(gpu.device), x.to(gpu.device).int(), V, sparse=True)
    n = ids.numel()
    assert torch.equal(got_ids[:n].cpu(), ids) and (got_ids[n:] == -1).all()
    assert torch.equal(rows[:n].cpu(), want[ids]) and not rows[n:].any()
    bad = x.clone()
    bad[T // 2] = V
    for sparse in (False, True):
        with pytest.raises(ValueError, match="outside"):
            mc.embedding_grad(gr.to(gpu.device), bad.to(gpu.device), V, sparse=sparse)


def test_gradients_written_anywhere(gpu):
    """Outputs that start off a 16-byte boundary, between values that stay."""
    lib = _lib.load()
    g = cases.gen(13)
    V, D = 37, 5
    for T in (300, 20000):
        x = ref.make_nodes(g, (T,), V, 0.2).to(gpu.device)
        gr = torch.randn(T, D, generator=g).to(torch.bfloat16).to(gpu.device)
        want = mc.embedding_grad(gr, x, V)
        need = lib.mlxc_embedding_grad_workspace_bytes(V, D, T, 0)
        work = torch.empty(need // 8 + 1, dtype=torch.int64, device=gpu.device)
        for skip in range(9):
            buf = torch.full((skip + V * D + 9,), 7.0, dtype=torch.bfloat16, device=gpu.device)
            assert lib.mlxc_embedding_grad(gr.data_ptr(), D, 1, x.data_ptr(), T, 0, V, 1.0, 0, None,
                                           buf.data_ptr() + 2 * skip, 1, work.data_ptr(), need,
                                           torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(buf[skip:skip + V * D].reshape(V, D), want)
            assert (buf[:skip] == 7).all() and (buf[skip + V * D:] == 7).all()


@pytest.mark.parametrize("dtype,D", [(torch.float32, 128), (torch.bfloat16, 128),
                                     (torch.float16, 100), (torch.bfloat16, 64)])
def test_window_scores_large(gpu, dtype, D):
    g = cases.gen(D)
    V, N, M, C = 3000, 3001, 81, 10
    w = torch.randn(V, D, generator=g).to(dtype).to(gpu.device)
    x = ref.make_nodes(g, (N, M), V, 0.01, 0.05).to(gpu.device)
    W = M - C + 1
    r = torch.where((x >= 0).unsqueeze(-1), w.double()[x.clamp(min=0)], 0.0)
    got = mc.window_scores(w, x, C, scale=0.3)
    for k in range(1, C):
        p = r[:, :W] * r[:, k:k + W]
        bound = 1.01 * (D + 8) * ref.U32 * p.abs().sum(-1) * 0.3
        assert float(((got[:, :, k - 1].double() - p.sum(-1) * 0.3).abs() - bound).max()) <= 0
    gr = torch.randn(got.shape, generator=g).to(gpu.device)
    du, size = torch.zeros_like(r), torch.zeros_like(r)
    for k in range(1, C):
        d = gr[:, :, k - 1].double().unsqueeze(-1) * ((x[:, :W] >= 0) & (x[:, k:k + W] >= 0)).unsqueeze(-1)
        for a, b in ((slice(0, W), slice(k, k + W)), (slice(k, k + W), slice(0, W))):
            du[:, a] += d * r[:, b]
            size[:, a] += (d * r[:, b]).abs()
    keep = (x.reshape(-1) >= 0).cpu()
    at = x.reshape(-1).cpu()[keep]
    sizes = sum_by_node(size.reshape(-1, D).cpu()[keep], at, V)
    total = sum_by_node(du.reshape(-1, D).cpu()[keep], at, V)
    n = torch.bincount(at, minlength=V).double().unsqueeze(1) * 2 * C
    value, bound = ref.stored(total * 0.3, (n + 4) * ref.U32 * sizes * 0.3, dtype)
    out = mc.window_scores_grad(gr, w, x, C, scale=0.3)
    assert float(((out.cpu().double() - value).abs() - bound).max()) <= 0
    ids, rows = mc.window_scores_grad(gr, w, x, C, scale=0.3, sparse=True)
    have = ids >= 0
    assert torch.equal(out[ids[have]], rows[have])
    assert torch.equal(mc.window_scores_grad(gr, w, x, C, scale=0.3), out)


def test_long_table_offsets(gpu):
    # rows past 2^32 bytes and 2^31 values of a table
    V, D = (1 << 25) + 3, 64
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=gpu.device)
    x = torch.tensor([[0, V - 1, V - 2, 1 << 24, V - 1]], device=gpu.device)
    w[x[0]] = torch.arange(1, 6, device=gpu.device).to(torch.bfloat16).unsqueeze(1)
    rows = mc.embedding(w, x)
    assert rows[0, :, 5].tolist() == [1.0, 5.0, 3.0, 4.0, 5.0]
    s = mc.window_scores(w, x, 2)
    assert s.flatten().tolist() == [64 * 5.0, 64 * 15.0, 64 * 12.0, 64 * 20.0]
    g = mc.embedding_grad(rows, x, V)
    assert g[V - 1].tolist() == [10.0] * D and g[V - 2].tolist() == [3.0] * D
    ids, r = mc.window_scores_grad(torch.ones_like(s), w, x, 2, sparse=True)
    assert ids.tolist() == [0, 1 << 24, V - 2, V - 1, -1]
    assert r[:, 0].tolist() == [5.0, 8.0, 9.0, 8.0, 0.0]


# ---- ways to call


def test_bad_nodes_raise_and_unchecked_ones_are_none(gpu):
    w = torch.randn(50, 16, device=gpu.device)
    x = torch.randint(0, 50, (6, 7), device=gpu.device)
    x[3, 4], x[0, 0] = 50, -2
    y = torch.where((x >= 0) & (x < 50), x, -1)
    for f in (lambda n, **k: mc.embedding(w, n, **k), lambda n, **k: mc.window_scores(w, n, 3, **k),
              lambda n, **k: mc.embedding_grad(w[:1].expand(6, 7, 16), n, 50, **k),
              lambda n, **k: mc.window_scores_grad(torch.ones(6, 5, 2, device=gpu.device), w, n, 3,
                                                   **k)):
        with pytest.raises(ValueError, match="outside"):
            f(x)
        assert torch.equal(f(x, check=False), f(y))
        f(y)  # the status of one call does not stay for the next


def test_other_streams(gpu):
    g = cases.gen(9)
    w = torch.randn(5000, 64, generator=g).to(gpu.device)
    x = ref.make_nodes(g, (800, 20), 5000, 0.1).to(gpu.device)
    s = mc.window_scores(w, x, 5)
    d = mc.window_scores_grad(s, w, x, 5)
    e = mc.embedding_grad(mc.embedding(w, x), x, 5000)
    p = mc.preference_loss_grad(s[:400], s[400:])
    side = torch.cuda.Stream()
    s2 = mc.window_scores(w, x, 5, stream=side, check=False)
    d2 = mc.window_scores_grad(s, w, x, 5, stream=side, check=False)
    e2 = mc.embedding_grad(mc.embedding(w, x, stream=side), x, 5000, stream=side)
    side.synchronize()
    p2 = mc.preference_loss_grad(s[:400], s[400:], stream=side)
    side.synchronize()
    assert torch.equal(s, s2) and torch.equal(d, d2) and torch.equal(e, e2)
    assert all(torch.equal(a, b) for a, b in zip(p, p2))
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        s3 = mc.window_scores(w, x, 5)
    assert torch.equal(s, s3)


def test_graph_replays(gpu):
    """A step in a HIP graph, replayed with new inputs between eager calls."""
    g = cases.gen(10)
    w = torch.randn(3000, 32, generator=g).to(gpu.device)
    walks = [ref.make_nodes(g, (700, 12), 3000, 0.05, 0.1).to(gpu.device) for _ in range(4)]
    x = walks[0].clone()

    def step(n):
        s = mc.window_scores(w, n, 4, check=False)
        loss, rewards, dc, dr = mc.preference_loss_grad(s[:350], s[350:], beta=0.3)
        grad = mc.window_scores_grad(torch.cat([dc, dr]), w, n, 4, check=False)
        ids, rows = mc.embedding_grad(mc.embedding(w, n, check=False), n, 3000, sparse=True,
                                      check=False)
        return s, loss, rewards, grad, ids, rows

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x)
    for n in walks * 2:
        x.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = step(n)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_broadcast_gradients_and_cpu_inputs(gpu):
    g = cases.gen(11)
    w = torch.randn(30, 8, generator=g)
    x = ref.make_nodes(g, (5, 6), 30, 0.2)
    p = w.to(gpu.device).requires_grad_()
    mc.embedding(p, x).sum().backward()  # the gradient is one value, expanded
    n = torch.bincount(x[x >= 0], minlength=30).float()
    assert torch.equal(p.grad.cpu(), n.unsqueeze(1).expand(30, 8))
    host = w.clone().requires_grad_()  # inputs on the CPU are copied, the gradient comes back
    mc.window_scores(host, x, 3, stream="cuda").sum().backward()
    other = w.to(gpu.device).requires_grad_()
    mc.window_scores(other, x.to(gpu.device), 3).sum().backward()
    assert host.grad.device.type == "cpu" and torch.equal(host.grad, other.grad.cpu())


def test_workspace_of_exactly_the_size_asked_for(gpu):
    lib = _lib.load()
    g = cases.gen(12)
    V, T, D = 700, 9001, 24
    x = ref.make_nodes(g, (T,), V, 0.1, 0.5).to(gpu.device)
    gr = torch.randn(T, D, generator=g).to(gpu.device)
    want = mc.embedding_grad(gr, x, V)
    need = lib.mlxc_embedding_grad_workspace_bytes(V, D, T, 0)
    for fill in (0, 0xAB):
        buf = torch.full((need + 512,), fill, dtype=torch.uint8, device=gpu.device)
        out = torch.empty(V, D, device=gpu.device)
        assert lib.mlxc_embedding_grad(gr.data_ptr(), D, 0, x.data_ptr(), T, 0, V, 1.0, 0, None,
                                       out.data_ptr(), 0, buf.data_ptr(), need, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (buf[need:] == fill).all()
    assert lib.mlxc_embedding_grad(gr.data_ptr(), D, 0, x.data_ptr(), T, 0, V, 1.0, 0, None,
                                   out.data_ptr(), 0, buf.data_ptr(), need - 1, None) == -1


def test_example_and_the_host_twins_agree(gpu):
    """examples/train_embeddings.py on the GPU: the first losses are the host
    twins' to what float32 adds in a step, and it learns."""
    import importlib.util
    import os

    from conftest import REPO
    spec = importlib.util.spec_from_file_location(
        "train_embeddings", os.path.join(REPO, "examples", "train_embeddings.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    kw = dict(nodes=1000, steps=40, batch=500, labelled=0.05, log=lambda *a: None)
    first, last, right = example.train(device="cuda", **kw)
    host, _, _ = example.train(device="cpu", **{**kw, "steps": 3})
    assert all(abs(a - b) < 1e-5 for a, b in zip(first, host))
    assert max(last) < 0.6 and right > 0.6


# ---- the compiled path and the Python layer


def test_compiled_path_and_python_layer_agree(gpu, monkeypatch):
    from mlx_cluster_amd import training
    if training._fast is None:
        pytest.skip("the compiled binding is not built")
    g = cases.gen(14)
    w = torch.randn(900, 48, generator=g).to(torch.bfloat16).to(gpu.device)
    x = ref.make_nodes(g, (60, 9), 900, 0.1).to(gpu.device)
    bad = x.clone()
    bad[5, 5] = 900
    sc = mc.window_scores(w, x, 4)
    m = torch.rand(sc.shape, generator=g).to(gpu.device) < 0.7
    calls = [
        lambda: mc.embedding(w, x, scale=2.0), lambda: mc.embedding(w, x.int(), check=False),
        lambda: mc.embedding_grad(mc.embedding(w, x), x, 900),
        lambda: mc.embedding_grad(mc.embedding(w, x), x, 900, sparse=True, check=False),
        lambda: mc.window_scores(w, x, 4), lambda: mc.window_scores(w, x),
        lambda: mc.window_scores_grad(sc, w, x, 4), lambda: mc.window_scores_grad(sc, w, x, 4, sparse=True),
        lambda: mc.preference_loss_grad(sc, sc.flip(0), beta=0.3),
        lambda: mc.preference_loss_grad(sc, sc.flip(0), sc * 0.5, None, chosen_mask=m, normalize=True,
                                        reduction="sum", label_smoothing=0.1),
    ]
    refusals = [
        lambda: mc.embedding(w, bad), lambda: mc.embedding_grad(mc.embedding(w, x), bad, 900),
        lambda: mc.window_scores(w, bad, 4), lambda: mc.window_scores_grad(sc, w, bad, 4),
        lambda: mc.window_scores(w, x, 10), lambda: mc.embedding(w.t(), x.float()),
        lambda: mc.embedding_grad(mc.embedding(w, x), x[:5], 900),
        lambda: mc.preference_loss_grad(sc, sc[:3]), lambda: mc.preference_loss_grad(sc, sc, sc[:3]),
    ]

    def outcome(call):
        try:
            out = call()
            return out if isinstance(out, tuple) else (out,)
        except (TypeError, ValueError) as e:
            return type(e), str(e)

    fast = [outcome(c) for c in calls + refusals]
    monkeypatch.setattr(training, "_fast", None)
    slow = [outcome(c) for c in calls + refusals]
    for a, b in zip(fast, slow):
        assert len(a) == len(b)
        for p, q in zip(a, b):
            assert torch.equal(p, q) if isinstance(p, torch.Tensor) else p == q
    assert all(isinstance(a[0], type) for a in fast[len(calls):])


def test_non_finite_rows_stay_where_they_are(gpu):
    """A row of infinities or NaN reaches the pairs it is in and no others."""
    g = cases.gen(15)
    for dtype in cases.FLOATS:
        for value in (float("nan"), float("inf")):
            for C in (3, 20):
                w = torch.randn(200, 64, generator=g)
                w[7] = value
                x = torch.randperm(199, generator=g)[:120].reshape(2, 60)
                x[x == 7] = 199
                x[0, 30] = 7
                w = w.to(dtype)
                s = mc.window_scores(w.to(gpu.device), x.to(gpu.device), C).cpu()
                hit = torch.zeros(s.shape, dtype=torch.bool)
                for j in range(60 - C + 1):
                    for k in range(1, C):
                        hit[0, j, k - 1] = j == 30 or j + k == 30
                assert not torch.isfinite(s[hit]).any() and torch.isfinite(s[~hit]).all()
                gr = torch.randn(s.shape, generator=g)
                d = mc.window_scores_grad(gr.to(gpu.device), w.to(gpu.device), x.to(gpu.device),
                                          C).cpu()
                near = set(x[0, max(0, 30 - C + 1):30 + C].tolist()) - {7}
                odd = {v for v in range(200) if not torch.isfinite(d[v].float()).all()}
                assert odd <= near and (odd == near or C > 3)
                clean = w.clone()
                clean[7] = 0
                e = mc.window_scores_grad(gr.to(gpu.device), clean.to(gpu.device),
                                          x.to(gpu.device), C).cpu()
                ok = torch.tensor([v not in near for v in range(200)])
                u = ref.ROUND[dtype][0] * 4
                assert ((d[ok].float() - e[ok].float()).abs() <= u * (1 + e[ok].float().abs()) * 10).all()


def test_largest_width_and_misaligned_arrays(gpu):
    """Rows that start at any element, wide rows, short and long preference rows off
    their alignment."""
    g = cases.gen(16)
    for dtype in cases.FLOATS:
        for skip in (1, 2, 3):
            flat = torch.randn(skip + 50 * 40, generator=g).to(dtype).to(gpu.device)
            w = flat[skip:].reshape(50, 40)
            x = ref.make_nodes(g, (6, 11), 50, 0.1).to(gpu.device)
            same = w.clone()
            assert torch.equal(mc.embedding(w, x), mc.embedding(same, x))
            a, b = mc.window_scores(w, x, 5), mc.window_scores(same, x, 5)
            assert torch.equal(a, b)
            assert torch.equal(mc.window_scores_grad(a, w, x, 5), mc.window_scores_grad(a, same, x, 5))
            rows = torch.randn(skip + 66 * 40, generator=g).to(dtype).to(gpu.device)[skip:].reshape(6, 11, 40)
            assert torch.equal(mc.embedding_grad(rows, x, 50), mc.embedding_grad(rows.clone(), x, 50))
            for T in (9, 100, 1500):
                v = torch.randn(skip + 12 * T, generator=g).to(dtype).to(gpu.device)[skip:].reshape(12, T)
                got = mc.preference_loss_grad(v, v.flip(0), beta=0.01, reduction="sum")
                want = mc.preference_loss_grad(v.clone(), v.flip(0), beta=0.01, reduction="sum")
                for p, q in zip(got, want):
                    assert torch.allclose(p.float(), q.float(), rtol=1e-5 + 4 * ref.ROUND[p.dtype][0],
                                          atol=1e-6)
    w = torch.randn(20, 5000, generator=g)
    x = ref.make_nodes(g, (3, 20), 20, 0.1)
    for C in (4, 20):
        want, bound = ref.window_scores(w, x, C, 1.0)
        ref.close(mc.window_scores(w.to(gpu.device), x.to(gpu.device), C), want, bound)


@pytest.mark.parametrize("dtype", cases.FLOATS)
@pytest.mark.parametrize("D", [33, 64, 260])
def test_one_window_gradients_by_hand(gpu, dtype, D):
    """Walks of one window: pairs without a node count nothing, whatever their gradients hold;
    a row of NaN reaches the rows it is paired with.  Every product is exact."""
    g = cases.gen(16, D)
    V, C = 30, 12
    w = torch.randint(-4, 5, (V, D), generator=g).float()
    w[29] = float("nan")
    x = torch.arange(2 * C).reshape(2, C)
    x[0, 3], x[0, 7], x[0, 9] = -1, V, 29
    x = torch.cat([x, x[1:2]])
    x[2, 0] = -1  # no first node: nothing
    gr = torch.randint(-2, 3, (3, 1, C - 1), generator=g).float()
    gr[0, 0, 2], gr[0, 0, 6], gr[2] = float("nan"), float("inf"), float("nan")
    gr[0, 0, 8] = 1
    want = torch.zeros(V, D)
    for n in range(2):
        for k in range(1, C):
            a, b = int(x[n, 0]), int(x[n, k])
            if 0 <= b < V:
                want[a] += gr[n, 0, k - 1] * w[b]
                want[b] += gr[n, 0, k - 1] * w[a]
    got = mc.window_scores_grad(gr.to(gpu.device), w.to(dtype).to(gpu.device), x.to(gpu.device), C,
                                check=False).cpu().float()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
