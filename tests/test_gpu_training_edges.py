"""The training operators' kernels at row sizes, table sizes and ways to call
that lie between those of test_gpu_training.py."""
import threading
import time
from types import SimpleNamespace

import pytest
import torch

import mlx_cluster_amd as mc
import train_cases as cases
import train_edges as edges
import train_reference as ref
from mlx_cluster_amd import _lib

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


def written(V, D, T, dtype, sparse, x, g, skip=0):
    """The gradient's rows through the C ABI, in memory that held sevens."""
    lib = _lib.load()
    flags = _lib.MLXC_GRAD_SPARSE if sparse else 0
    rows = min(V, T) if sparse else V
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    buf = torch.full((skip + rows * D + 8,), 7.0, dtype=dtype, device=x.device)
    ids = torch.full((rows + 1,), 7, dtype=torch.int64, device=x.device)
    need = lib.mlxc_embedding_grad_workspace_bytes(V, D, T, flags)
    work = torch.empty(need // 8 + 1, dtype=torch.int64, device=x.device)
    rc = lib.mlxc_embedding_grad(
        g.data_ptr(), D, code, x.data_ptr(), T, 0, V, 1.0, flags, ids.data_ptr() if sparse else None,
        buf.data_ptr() + skip * buf.element_size(), code, work.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, _lib.last_error()
    assert (buf[:skip] == 7).all() and (buf[skip + rows * D:] == 7).all() and int(ids[-1]) == 7
    return buf[skip:skip + rows * D].reshape(rows, D), ids[:-1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [0, 20000, 70000])
def test_every_byte_of_a_gradient_is_written(gpu, T, dtype):
    """No node at all: every size of the rows up to two packs, and around whole pages, at every
    start that the type allows."""
    x = torch.full((max(T, 1),), -1, device=gpu.device)
    g = torch.ones(max(T, 1), device=gpu.device).to(dtype)
    esz = g.element_size()
    sizes = list(range(1, 25)) + [4096 * k // esz + d for k in range(1, 9) for d in range(-5, 6)]
    for n in sizes:
        for skip in (0, n % (16 // esz)):
            out, _ = written(n, 1, T, dtype, False, x, g, skip)
            assert not out.any(), (n, skip, out.nonzero().flatten().tolist()[:4])
        if T:
            out, ids = written(n, 1, T, dtype, True, x, g)
            assert not out.any() and (ids == -1).all(), n


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("V,D,T,dtype", [
    (1025, 1, 20000, torch.float32), (3, 1, 20000, torch.float32), (683, 3, 20000, torch.float32),
    (41, 50, 20000, torch.bfloat16), (82, 50, 20000, torch.bfloat16), (41, 100, 70000, torch.bfloat16),
    (1229, 10, 20000, torch.bfloat16), (41, 50, 20000, torch.float32)])
def test_rows_that_no_place_visits_are_zeros(gpu, V, D, T, dtype, sparse):
    x = torch.arange(T, device=gpu.device) % (V - 2)  # the last two rows: none
    g = torch.ones(T, D, device=gpu.device).to(dtype)
    out, ids = written(V, D, T, dtype, sparse, x, g)
    n = torch.bincount(x, minlength=V).to(dtype)
    assert torch.equal(out, n.unsqueeze(1).expand(V, D))
    if sparse:
        assert ids.tolist() == [*range(V - 2), -1, -1]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_dual_tensors_are_refused(gpu, grad_mode, requires_grad):
    edges.check_dual_tensors(gpu, grad_mode, requires_grad)


def keep_busy(stream, device):
    """Some milliseconds of work on `stream`."""
    with torch.cuda.stream(stream):
        a = torch.ones(4096, 4096, device=device)
        for _ in range(4):
            a = a @ a * 1e-4
    return a


@pytest.mark.parametrize("sparse", [False, True])
def test_backward_on_another_stream(gpu, sparse):
    """What autograd does with a gradient comes after the kernels that make it, whatever stream
    the call named and however long that stream is busy."""
    g = cases.gen(21)
    table = torch.randn(3000, 48, generator=g)
    x = ref.make_nodes(g, (900, 14), 3000, 0.05, 0.1).to(gpu.device)
    other = ref.make_nodes(g, (900, 14), 3000, 0.0).to(gpu.device)
    side = torch.cuda.Stream()

    def step(stream, device):
        # dense: one table in three calls, whose gradients autograd adds up; coalesced: one each
        leaf = lambda: table.clone().to(device).requires_grad_()
        leaves = [leaf() for _ in range(3)] if sparse else [leaf()] * 3
        torch.cuda.synchronize()
        kw = dict(sparse_grad=sparse, stream=stream)
        pos = mc.window_scores(leaves[0], x, 5, **kw)
        neg = mc.window_scores(leaves[1], other, 5, **kw)
        rows = mc.embedding(leaves[2], x, scale=0.5, **kw)
        torch.cuda.synchronize()
        loss = mc.preference_loss(pos, neg, beta=0.5, stream=stream)
        torch.cuda.synchronize()
        busy = keep_busy(side, gpu.device)
        (loss * 7.0 + (rows * rows).sum() * 0.01).backward()
        return [p.grad.to_dense().cpu() if sparse else p.grad.cpu() for p in leaves]

    want = step(None, gpu.device)
    for device in (gpu.device, gpu.device, "cpu"):  # a table on the CPU gets its gradient there
        assert all(torch.equal(a, b) for a, b in zip(step(side, device), want))


@pytest.mark.parametrize("mask", [False, True])
def test_preference_backward_on_another_stream(gpu, mask):
    g = cases.gen(22)
    values = [torch.randn(500, n, generator=g).to(gpu.device) for n in (70, 9)]
    masks = [(torch.rand(v.shape, generator=g) < 0.7).to(gpu.device) if mask else None
             for v in (values[0].cpu(), values[1].cpu())]
    side = torch.cuda.Stream()

    def step(stream):
        leaves = [v.clone().requires_grad_() for v in values]
        torch.cuda.synchronize()
        loss = mc.preference_loss(leaves[0] * 2.0, leaves[1] * 3.0, chosen_mask=masks[0],
                                  rejected_mask=masks[1], stream=stream)
        if stream is not None:
            stream.synchronize()
            busy = keep_busy(stream, gpu.device)
        loss.backward()
        return [v.grad.cpu() for v in leaves]

    want = step(None)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(side), want))


def test_sizes_past_32_bits(gpu):
    edges.check_sizes_past_32_bits(gpu)


def test_other_threads_run_while_a_checked_call_waits(gpu):
    """A checked call waits for all that is queued before it; it does not hold the interpreter."""
    g = cases.gen(23)
    w = torch.randn(500, 16, generator=g).to(gpu.device)
    x = ref.make_nodes(g, (40, 8), 500, 0.1).to(gpu.device)
    grad = mc.embedding(w, x)
    scores = mc.window_scores(w, x, 3)
    a = torch.ones(8192, 8192, device=gpu.device)
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.001)

    thread = threading.Thread(target=tick)
    thread.start()
    try:
        for call in (lambda: mc.embedding(w, x), lambda: mc.embedding_grad(grad, x, 500),
                     lambda: mc.window_scores(w, x, 3), lambda: mc.window_scores_grad(scores, w, x, 3)):
            call()
            torch.cuda.synchronize()
            for _ in range(10):  # some tens of milliseconds
                a = a @ a * 1e-4
            t0 = time.perf_counter()
            call()
            t1 = time.perf_counter()
            assert t1 - t0 > 0.02  # it waited
            during = [t for t in ticks if t0 < t < t1]
            assert len(during) >= 5
    finally:
        stop.set()
        thread.join()


def test_non_finite_rows_reach_every_place_they_are_paired_with(gpu):
    """The gradient of every place that is in a pair with a row of NaN or infinities is one too,
    over several tiles of places, and no other is."""
    g = cases.gen(15)
    for dtype in cases.FLOATS:
        for value in (float("nan"), float("inf")):
            for M, C, at in ((60, 20, 30), (60, 3, 30), (90, 32, 47), (70, 17, 5), (61, 32, 60)):
                w = torch.randn(200, 64, generator=g)
                w[7] = value
                w = w.to(dtype)
                x = torch.randperm(199, generator=g)[:M].unsqueeze(0)
                x[x == 7] = 199
                x[0, at] = 7
                gr = 1.0 + torch.rand(1, M - C + 1, C - 1, generator=g)
                pairs = {o for o in range(M)
                         if 0 < abs(o - at) < C and min(o, at) < M - C + 1}
                d = mc.window_scores_grad(gr.to(gpu.device), w.to(gpu.device), x.to(gpu.device),
                                          C).cpu()
                odd = {v for v in range(200) if not torch.isfinite(d[v].float()).all()}
                assert odd == {int(x[0, o]) for o in pairs}


@pytest.mark.parametrize("D,dtype", [(256, torch.float32), (260, torch.bfloat16), (33, torch.float16)])
@pytest.mark.parametrize("hub", [0.0, 0.5, 1.0])
def test_short_lists_of_hubs(gpu, hub, D, dtype):
    """The largest list that one launch takes, all or half of it one node, with wide rows of
    values that round."""
    T, V = 16384, 700
    g = cases.gen(T, D)
    x = ref.make_nodes(g, (T,), V, 0.0, hub)
    gr = torch.randn(T, D, generator=g).to(dtype)
    got = mc.embedding_grad(gr.to(gpu.device), x.to(gpu.device), V).cpu()
    total = torch.zeros(V, D, dtype=torch.float64).index_add_(0, x, gr.double())
    size = torch.zeros(V, D, dtype=torch.float64).index_add_(0, x, gr.double().abs())
    n = torch.bincount(x, minlength=V).double().unsqueeze(1)
    ref.close(got, *ref.stored(total, (n + 4) * ref.U32 * size, dtype))
