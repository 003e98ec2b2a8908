"""Training node embeddings on walks (libmlxc.so, include/mlxc_train.h).

The reference stops at the walks (/root/reference/random_walks/
BiasedRandomWalk.cpp:96).  What trains on them next is here: rows of a table by
node (`embedding`), the scores of skip-gram windows (`window_scores`), a loss
of preferred against other windows or sequences (`preference_loss`), and their
gradients (`embedding_grad`, `window_scores_grad`, `preference_loss_grad`).

The first three are differentiable by torch's autograd (once, backward; dual
tensors raise NotImplementedError); the `_grad` functions are the same kernels
for programs that write their own step.  A node of -1 is no node: its row reads
as zeros and takes no gradient.  Sums are made in 32 bits or more and rounded
once; the same call gives the same bits every time.  On the GPU the operators
run in HIP kernels, with stream='cpu' in host twins that follow the same
formulas with 64-bit sums.
"""
from __future__ import annotations

import ctypes
import math
import numbers
from typing import Optional, Tuple, Union

import numpy as np
import torch

from . import _lib
from .walks import (_check_stream_arg, _fast, _enter_side_stream, _leave_side_stream, _on, _on_cpu,
                    _on_device, _ptr, _resolve_device, _side_stream, _stream_handle, _workspace)

_FLOATS = {torch.float32: _lib.MLXC_FLOAT32, torch.bfloat16: _lib.MLXC_BFLOAT16,
           torch.float16: _lib.MLXC_FLOAT16}
_NODES = {torch.int64: _lib.MLXC_OUT_INT64, torch.int32: _lib.MLXC_OUT_INT32}

# The library's widest row, and the sizes that it takes as 32-bit numbers: refused
# here, before they are cut to 32 bits on their way there.
_MAX_DIM = 65536
_MAX_SIZE = 2**31 - 1

Grad = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


# ---------------------------------------------------------------- arguments

def _tensor(x, types, name: str) -> torch.Tensor:
    if isinstance(x, np.ndarray):
        x = torch.from_numpy(x)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or numpy.ndarray, got {type(x)!r}")
    if x.dtype not in types:
        names = ", ".join(str(t) for t in types)
        raise TypeError(f"{name} must have dtype {names}, got {x.dtype}")
    return x


def _number(x, name: str) -> float:
    if isinstance(x, bool) or not isinstance(x, numbers.Real):
        raise TypeError(f"{name} must be a number")
    return float(x)


def _int(x, name: str) -> int:
    if isinstance(x, bool) or not isinstance(x, numbers.Integral):
        raise TypeError(f"{name} must be an int")
    return int(x)


def _table(weight) -> torch.Tensor:
    weight = _tensor(weight, _FLOATS, "weight")
    if weight.dim() != 2 or weight.shape[1] < 1:
        raise ValueError("weight must be a 2-D [num_nodes, dim >= 1] tensor")
    _check_dim(weight.shape[1])
    return weight


def _check_dim(dim: int) -> None:
    if dim > _MAX_DIM:
        raise ValueError(f"dim must lie in [1, {_MAX_DIM}], got {dim}")


def _rows_on(weight: torch.Tensor, device: torch.device) -> torch.Tensor:
    """The table on `device`, its rows' values next to each other; rows may lie
    any stride apart (a table is not copied for its row stride)."""
    weight = weight.detach()
    if weight.device != device:
        weight = weight.to(device)
    D = weight.shape[1]
    if (weight.stride(1) == 1 or D == 1) and (weight.shape[0] < 2 or weight.stride(0) >= D):
        return weight
    return weight.contiguous()


def _row_stride(weight: torch.Tensor) -> int:
    return weight.stride(0) if weight.shape[0] > 1 else max(weight.stride(0), weight.shape[1])


def _walks(walks, context_size) -> Tuple[torch.Tensor, int]:
    walks = _tensor(walks, _NODES, "walks")
    if walks.dim() != 2 or walks.shape[1] < 2:
        raise ValueError("walks must be a 2-D [N, nodes >= 2] tensor")
    if walks.shape[1] > _MAX_SIZE:
        raise ValueError(f"walks of at most {_MAX_SIZE} nodes, got {walks.shape[1]}")
    C = walks.shape[1] if context_size is None else _int(context_size, "context_size")
    if not 2 <= C <= min(32, walks.shape[1]):
        raise ValueError("context_size must lie in [2, min(32, nodes per walk)]")
    return walks, C


def _out_dtype(out_dtype, default: torch.dtype) -> torch.dtype:
    if out_dtype is None:
        return default
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype!r}")
    return out_dtype


def _raise_bad(bits: int, what: str) -> None:
    if bits & _lib.MLXC_STATUS_BAD_NODE:
        raise ValueError(f"{what}: a node is outside [0, num_nodes) and not -1")


def _read_status(word: torch.Tensor, stream, what: str) -> None:
    if isinstance(stream, torch.cuda.Stream):
        stream.synchronize()
    _raise_bits = int(word[0].item())
    _raise_bad(_raise_bits, what)


def _plain(stream, number, *tensors) -> bool:
    """Whether the compiled path (csrc/torch_training.cpp) may take a call: it
    looks at the tensors itself, and leaves what it does not take to the code
    below."""
    return (_fast is not None and stream is None and type(number) is float and
            all(isinstance(t, torch.Tensor) for t in tensors))


def _plain_int(x) -> bool:
    return x is None or (type(x) is int and 0 < x <= _MAX_SIZE)


class _Launch:
    """A call's device, stream handle and side stream; `with` it, kernels
    launch there and every tensor given to `uses` is held for them."""

    def __init__(self, stream, tensors):
        self.stream = stream
        self.device = _resolve_device(stream, tensors)
        self.handle = _stream_handle(stream, self.device)
        self.side = _side_stream(stream, self.device)
        self.tensors = ()

    def uses(self, *tensors):
        self.tensors = tensors
        return self

    def __enter__(self):
        _enter_side_stream(self.side, self.device)
        self.on = _on_device(self.device)
        self.on.__enter__()
        return self

    def __exit__(self, *exc):
        self.on.__exit__(*exc)
        _leave_side_stream(self.side, *self.tensors)
        return False


def _join_side_stream(stream) -> None:
    """Torch's current stream waits for a backward's kernels on `stream`: autograd
    adds their results up and hands them on at once, and leaves no place for the
    caller to wait (as a forward call on another stream does)."""
    if isinstance(stream, torch.cuda.Stream):
        side = _side_stream(stream, stream.device)
        if side is not None:
            torch.cuda.current_stream(stream.device).wait_stream(side)


# ---------------------------------------------------------------- embedding

def _embedding(weight, nodes, scale: float, check: bool, stream) -> torch.Tensor:
    lib = _lib.load()
    V, D = weight.shape
    count = nodes.numel()
    if _on_cpu(stream):
        weight, nodes = _rows_on(weight, torch.device("cpu")), nodes.cpu().contiguous()
        out = torch.empty((*nodes.shape, D), dtype=weight.dtype)
        status = ctypes.c_int64(0)
        _lib.check(lib.mlxc_embedding_cpu(
            _ptr(weight), V, D, _row_stride(weight), _FLOATS[weight.dtype], _ptr(nodes), count,
            _NODES[nodes.dtype], scale, _ptr(out), ctypes.addressof(status)), "embedding")
        if check:
            _raise_bad(status.value, "embedding")
        return out
    run = _Launch(stream, (weight, nodes))
    weight, nodes = _rows_on(weight, run.device), _on(nodes, run.device)
    out = torch.empty((*nodes.shape, D), dtype=weight.dtype, device=run.device)
    word = _workspace(8, run.device) if check else None
    with run.uses(weight, nodes, out, word):
        rc = lib.mlxc_embedding(
            _ptr(weight), V, D, _row_stride(weight), _FLOATS[weight.dtype], _ptr(nodes), count,
            _NODES[nodes.dtype], scale, _ptr(out), _ptr(word), run.handle)
    _lib.check(rc, "embedding")
    if check:
        _read_status(word, stream, "embedding")
    return out


class _EmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, nodes, scale, sparse_grad, check, stream):
        ctx.save_for_backward(nodes)
        ctx.args = (weight.shape[0], weight.dtype, weight.device, scale, sparse_grad, stream)
        return _embedding(weight, nodes, scale, check, stream)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (nodes,) = ctx.saved_tensors
        V, dtype, device, scale, sparse_grad, stream = ctx.args
        g = _embedding_grad(grad, nodes, V, scale, sparse_grad, dtype, False, stream)
        _join_side_stream(stream)
        return _autograd_grad(g, V, device), None, None, None, None, None


def _autograd_grad(grad: Grad, V: int, device) -> torch.Tensor:
    """A gradient for autograd, on the weight's device; a coalesced one as a
    sparse tensor (without the padding: it reads the number of nodes back)."""
    if not isinstance(grad, tuple):
        return grad.to(device)
    ids, rows = grad
    keep = ids >= 0
    return torch.sparse_coo_tensor(ids[keep].unsqueeze(0), rows[keep], (V, rows.shape[1]),
                                   is_coalesced=True).to(device)


def _tracked(*tensors) -> bool:
    """Whether autograd has to see a call: one to record, or one of dual tensors,
    which the functions above refuse (they have no forward-mode derivative)."""
    return any((t.requires_grad and torch.is_grad_enabled()) or
               torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def embedding(weight, nodes, *, scale: float = 1.0, sparse_grad: bool = False, check: bool = True,
              stream=None) -> torch.Tensor:
    """Rows of a table by node, scaled: scale * weight[nodes], [*nodes.shape, dim].

    Args:
        weight: [num_nodes, dim] float32, bfloat16 or float16; rows may lie any
            stride apart.  Differentiable.
        nodes: int64 or int32 of any shape: walks, windows, edge ids.  -1 is no
            node (the edge id of a step that stayed): a row of zeros.
        scale: factor of every row (for instance sqrt(dim)).
        sparse_grad: autograd's gradient as a coalesced sparse tensor.
        check: synchronise once and raise ValueError on other nodes outside
            [0, num_nodes); with False they read as zeros too, and the call
            stays asynchronous.
        stream: as in random_walk ('cpu' runs the host twin).
    """
    if _plain(stream, scale, weight, nodes) and not sparse_grad:
        res = _fast.embedding(weight, nodes, scale, bool(check))
        if res is not None:
            return res
    _check_stream_arg(stream)
    weight = _table(weight)
    nodes = _tensor(nodes, _NODES, "nodes")
    scale = _number(scale, "scale")
    if _tracked(weight):
        return _EmbeddingFunction.apply(weight, nodes, scale, bool(sparse_grad), check, stream)
    return _embedding(weight, nodes, scale, check, stream)


def _grad_buffers(V: int, D: int, count: int, sparse: bool, dtype, device):
    rows = min(count, V) if sparse else V
    out = torch.empty((rows, D), dtype=dtype, device=device)
    ids = torch.empty(rows, dtype=torch.int64, device=device) if sparse else None
    return ids, out, _lib.MLXC_GRAD_SPARSE if sparse else 0


def _embedding_grad(grad, nodes, V: int, scale: float, sparse: bool, out_dtype, check: bool,
                    stream) -> Grad:
    lib = _lib.load()
    D = grad.shape[-1]
    count = nodes.numel()
    grad = grad.detach()
    if _on_cpu(stream):
        grad, nodes = grad.cpu().contiguous(), nodes.cpu().contiguous()
        ids, out, flags = _grad_buffers(V, D, count, sparse, out_dtype, torch.device("cpu"))
        status = ctypes.c_int64(0)
        _lib.check(lib.mlxc_embedding_grad_cpu(
            _ptr(grad), D, _FLOATS[grad.dtype], _ptr(nodes), count, _NODES[nodes.dtype], V, scale,
            flags, _ptr(ids), _ptr(out), _FLOATS[out_dtype], ctypes.addressof(status)),
            "embedding_grad")
        if check:
            _raise_bad(status.value, "embedding_grad")
        return (ids, out) if sparse else out
    run = _Launch(stream, (grad, nodes))
    grad, nodes = _on(grad, run.device), _on(nodes, run.device)
    ids, out, flags = _grad_buffers(V, D, count, sparse, out_dtype, run.device)
    work = _grad_workspace(lib.mlxc_embedding_grad_workspace_bytes(V, D, count, flags), run.device,
                           "embedding_grad")
    with run.uses(grad, nodes, ids, out, work):
        rc = lib.mlxc_embedding_grad(
            _ptr(grad), D, _FLOATS[grad.dtype], _ptr(nodes), count, _NODES[nodes.dtype], V, scale,
            flags, _ptr(ids), _ptr(out), _FLOATS[out_dtype], work.data_ptr(), work.numel() * 8,
            run.handle)
    _lib.check(rc, "embedding_grad")
    if check:
        _read_status(work, stream, "embedding_grad")
    return (ids, out) if sparse else out


def _grad_workspace(nbytes: int, device, what: str) -> torch.Tensor:
    if nbytes == 0:
        raise ValueError(f"{what}: {_lib.last_error()}")
    return _workspace(nbytes, device)


def embedding_grad(grad, nodes, num_nodes: int, *, scale: float = 1.0, sparse: bool = False,
                   out_dtype: Optional[torch.dtype] = None, check: bool = True,
                   stream=None) -> Grad:
    """Gradient of `embedding` with respect to the table, by sorted nodes.

    Args:
        grad: [*nodes.shape, dim], the gradient of embedding's result.
        nodes, scale, check, stream: as in embedding.
        num_nodes: rows of the table.
        sparse: False returns the whole table's gradient [num_nodes, dim]; True
            returns (ids, rows): the nodes that occur, ascending, and their
            rows, both min(nodes, num_nodes) long: past the last node ids are
            -1 and rows zeros.  So their sizes do not depend on the values, and
            the call stays asynchronous with check=False.
        out_dtype: of the gradient (default: grad's).
    """
    if out_dtype is None and type(num_nodes) is int and 0 <= num_nodes <= _MAX_SIZE and \
            _plain(stream, scale, grad, nodes):
        res = _fast.embedding_grad(grad, nodes, num_nodes, scale, bool(sparse), bool(check))
        if res is not None:
            return res
    _check_stream_arg(stream)
    grad = _tensor(grad, _FLOATS, "grad")
    nodes = _tensor(nodes, _NODES, "nodes")
    scale = _number(scale, "scale")
    V = _int(num_nodes, "num_nodes")
    if not 0 <= V <= _MAX_SIZE:
        raise ValueError(f"num_nodes must lie in [0, {_MAX_SIZE}]")
    if grad.dim() != nodes.dim() + 1 or grad.shape[:-1] != nodes.shape or grad.shape[-1] < 1:
        raise ValueError("grad must have shape [*nodes.shape, dim >= 1]")
    _check_dim(grad.shape[-1])
    return _embedding_grad(grad, nodes, V, scale, bool(sparse), _out_dtype(out_dtype, grad.dtype),
                           check, stream)


# ---------------------------------------------------------------- windows

def _window_scores(weight, walks, C: int, scale: float, check: bool, stream) -> torch.Tensor:
    lib = _lib.load()
    V, D = weight.shape
    N, M = walks.shape
    shape = (N, M - C + 1, C - 1)
    if _on_cpu(stream):
        weight, walks = _rows_on(weight, torch.device("cpu")), walks.cpu().contiguous()
        out = torch.empty(shape, dtype=torch.float32)
        status = ctypes.c_int64(0)
        _lib.check(lib.mlxc_window_scores_cpu(
            _ptr(weight), V, D, _row_stride(weight), _FLOATS[weight.dtype], _ptr(walks), N, M, C,
            _NODES[walks.dtype], scale, _ptr(out), ctypes.addressof(status)), "window_scores")
        if check:
            _raise_bad(status.value, "window_scores")
        return out
    run = _Launch(stream, (weight, walks))
    weight, walks = _rows_on(weight, run.device), _on(walks, run.device)
    out = torch.empty(shape, dtype=torch.float32, device=run.device)
    word = _workspace(8, run.device) if check else None
    with run.uses(weight, walks, out, word):
        rc = lib.mlxc_window_scores(
            _ptr(weight), V, D, _row_stride(weight), _FLOATS[weight.dtype], _ptr(walks), N, M, C,
            _NODES[walks.dtype], scale, _ptr(out), _ptr(word), run.handle)
    _lib.check(rc, "window_scores")
    if check:
        _read_status(word, stream, "window_scores")
    return out


def _window_scores_grad(grad, weight, walks, C: int, scale: float, sparse: bool, out_dtype,
                        check: bool, stream) -> Grad:
    lib = _lib.load()
    V, D = weight.shape
    N, M = walks.shape
    grad = grad.detach()
    if _on_cpu(stream):
        host = torch.device("cpu")
        weight, walks, grad = _rows_on(weight, host), walks.cpu().contiguous(), _on(grad, host)
        ids, out, flags = _grad_buffers(V, D, N * M, sparse, out_dtype, host)
        status = ctypes.c_int64(0)
        _lib.check(lib.mlxc_window_scores_grad_cpu(
            _ptr(grad), _ptr(weight), V, D, _row_stride(weight), _FLOATS[weight.dtype],
            _ptr(walks), N, M, C, _NODES[walks.dtype], scale, flags, _ptr(ids), _ptr(out),
            _FLOATS[out_dtype], ctypes.addressof(status)), "window_scores_grad")
        if check:
            _raise_bad(status.value, "window_scores_grad")
        return (ids, out) if sparse else out
    run = _Launch(stream, (weight, grad, walks))
    weight, walks = _rows_on(weight, run.device), _on(walks, run.device)
    grad = _on(grad, run.device)
    ids, out, flags = _grad_buffers(V, D, N * M, sparse, out_dtype, run.device)
    work = _grad_workspace(lib.mlxc_window_scores_grad_workspace_bytes(V, D, N, M, C, flags),
                           run.device, "window_scores_grad")
    with run.uses(grad, weight, walks, ids, out, work):
        rc = lib.mlxc_window_scores_grad(
            _ptr(grad), _ptr(weight), V, D, _row_stride(weight), _FLOATS[weight.dtype],
            _ptr(walks), N, M, C, _NODES[walks.dtype], scale, flags, _ptr(ids), _ptr(out),
            _FLOATS[out_dtype], work.data_ptr(), work.numel() * 8, run.handle)
    _lib.check(rc, "window_scores_grad")
    if check:
        _read_status(work, stream, "window_scores_grad")
    return (ids, out) if sparse else out


class _WindowScoresFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, walks, C, scale, sparse_grad, check, stream):
        ctx.save_for_backward(weight, walks)
        ctx.args = (C, scale, sparse_grad, stream)
        return _window_scores(weight, walks, C, scale, check, stream)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, walks = ctx.saved_tensors
        C, scale, sparse_grad, stream = ctx.args
        g = _window_scores_grad(grad, weight, walks, C, scale, sparse_grad, weight.dtype, False,
                                stream)
        _join_side_stream(stream)
        return (_autograd_grad(g, weight.shape[0], weight.device),) + (None,) * 6


def window_scores(weight, walks, context_size: Optional[int] = None, *, scale: float = 1.0,
                  sparse_grad: bool = False, check: bool = True, stream=None) -> torch.Tensor:
    """Scores of the skip-gram windows of walks: float32 [N, W, C - 1].

    Entry [n, j, k - 1] is scale * <row of walk n's node j, row of its node
    j + k>, for the W = nodes - C + 1 windows of C = context_size nodes that
    context_windows cuts (here walk by walk, and without writing them).
    context_size None takes each row of `walks` as one window, for windows made
    elsewhere (negative_windows).  A pair with a node of -1 scores 0.

    weight, sparse_grad, check, stream: as in embedding; differentiable in
    weight.  walks: int64 or int32 [N, nodes], context_size in [2, min(32, nodes)].
    """
    if _plain(stream, scale, weight, walks) and _plain_int(context_size) and not sparse_grad:
        res = _fast.window_scores(weight, walks, context_size or 0, scale, bool(check))
        if res is not None:
            return res
    _check_stream_arg(stream)
    weight = _table(weight)
    walks, C = _walks(walks, context_size)
    scale = _number(scale, "scale")
    if _tracked(weight):
        return _WindowScoresFunction.apply(weight, walks, C, scale, bool(sparse_grad), check,
                                           stream)
    return _window_scores(weight, walks, C, scale, check, stream)


def window_scores_grad(grad, weight, walks, context_size: Optional[int] = None, *,
                       scale: float = 1.0, sparse: bool = False,
                       out_dtype: Optional[torch.dtype] = None, check: bool = True,
                       stream=None) -> Grad:
    """Gradient of `window_scores` with respect to the table.

    grad: float32 [N, W, C - 1], the gradient of the scores; what it holds at
    pairs with a node of -1 is not used.  weight, walks, context_size, scale,
    check, stream: as in window_scores.  sparse, out_dtype (default: weight's)
    and the result: as in embedding_grad.
    """
    if out_dtype is None and _plain_int(context_size) and \
            _plain(stream, scale, grad, weight, walks):
        res = _fast.window_scores_grad(grad, weight, walks, context_size or 0, scale, bool(sparse),
                                       bool(check))
        if res is not None:
            return res
    _check_stream_arg(stream)
    weight = _table(weight)
    walks, C = _walks(walks, context_size)
    scale = _number(scale, "scale")
    grad = _tensor(grad, (torch.float32,), "grad")
    shape = (walks.shape[0], walks.shape[1] - C + 1, C - 1)
    if tuple(grad.shape) != shape:
        raise ValueError(f"grad must have shape {list(shape)}, got {list(grad.shape)}")
    return _window_scores_grad(grad, weight, walks, C, scale, bool(sparse),
                               _out_dtype(out_dtype, weight.dtype), check, stream)


# ---------------------------------------------------------------- preference

class _Sides:
    """Checked arguments of a preference call."""

    def __init__(self, chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask,
                 beta, label_smoothing, normalize, reduction):
        self.values, self.refs, self.masks, self.shapes = [], [], [], []
        for name, x, ref, mask in (("chosen", chosen, ref_chosen, chosen_mask),
                                   ("rejected", rejected, ref_rejected, rejected_mask)):
            x = _tensor(x, _FLOATS, name)
            if x.dim() < 1:
                raise ValueError(f"{name} must have a pair dimension")
            self.shapes.append(x.shape)
            if ref is not None:
                ref = _tensor(ref, (x.dtype,), f"ref_{name}")
                if ref.shape != x.shape:
                    raise ValueError(f"ref_{name} must have {name}'s shape")
                ref = ref.detach()
            if mask is not None:
                mask = _tensor(mask, (torch.bool, torch.uint8), f"{name}_mask")
                if mask.shape != x.shape:
                    raise ValueError(f"{name}_mask must have {name}'s shape")
            self.values.append(x)
            self.refs.append(ref)
            self.masks.append(mask)
        if self.values[0].dtype != self.values[1].dtype:
            raise TypeError("chosen and rejected must have the same dtype")
        pairs = [s[:-1] if len(s) > 1 else s for s in self.shapes]
        if pairs[0] != pairs[1]:
            raise ValueError(f"chosen and rejected must hold the same pairs, got {list(pairs[0])} "
                             f"and {list(pairs[1])}")
        self.pairs = math.prod(pairs[0])
        self.lengths = [s[-1] if len(s) > 1 else 1 for s in self.shapes]
        self.beta = _number(beta, "beta")
        if not math.isfinite(self.beta):
            raise ValueError("beta must be finite")
        self.smoothing = _number(label_smoothing, "label_smoothing")
        if not 0.0 <= self.smoothing <= 1.0:
            raise ValueError("label_smoothing must lie in [0, 1]")
        if reduction not in ("mean", "sum"):
            raise ValueError("reduction must be 'mean' or 'sum'")
        self.flags = ((_lib.MLXC_PREFERENCE_NORMALIZE if normalize else 0) |
                      (_lib.MLXC_PREFERENCE_SUM if reduction == "sum" else 0))

    def on(self, device: torch.device) -> None:
        move = lambda ts: [None if t is None else _on(t.detach(), device) for t in ts]
        self.values, self.refs, self.masks = (move(t) for t in (self.values, self.refs, self.masks))

    def tensors(self):
        return [t for t in (*self.values, *self.refs, *self.masks) if t is not None]

    def structs(self, grads):
        return [_lib.PreferenceSide(_ptr(v), _ptr(r), _ptr(m), n, _ptr(g)) for v, r, m, n, g in
                zip(self.values, self.refs, self.masks, self.lengths, grads)]


def _preference(sides: _Sides, want_grads: bool, want_slopes: bool, stream):
    """(loss, rewards, slopes or None, grads)."""
    lib = _lib.load()
    on_cpu = _on_cpu(stream)
    if on_cpu:
        run, device = None, torch.device("cpu")
    else:
        run = _Launch(stream, sides.values)
        device = run.device
    sides.on(device)
    dtype = _FLOATS[sides.values[0].dtype]
    new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=device)
    loss, rewards = new(), new(2, sides.pairs)
    slopes = new(2, sides.pairs) if want_slopes else None
    grads = [torch.empty_like(v) if want_grads else None for v in sides.values]
    args = (sides.pairs, dtype, sides.beta, sides.smoothing, sides.flags, loss.data_ptr(),
            _ptr(rewards), _ptr(slopes))
    c, r = sides.structs(grads)
    if on_cpu:
        _lib.check(lib.mlxc_preference_loss_cpu(c, r, *args), "preference_loss")
        return loss, rewards, slopes, grads
    work = _workspace(lib.mlxc_preference_loss_workspace_bytes(sides.pairs), device)
    with run.uses(*sides.tensors(), loss, rewards, slopes, *grads, work):
        rc = lib.mlxc_preference_loss(c, r, *args, work.data_ptr(), work.numel() * 8, run.handle)
    _lib.check(rc, "preference_loss")
    return loss, rewards, slopes, grads


class _PreferenceFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, chosen, rejected, sides, stream):
        ctx.devices = (chosen.device, rejected.device)
        loss, rewards, slopes, _ = _preference(sides, False, True, stream)
        ctx.save_for_backward(slopes, *sides.masks)
        ctx.args = (sides.pairs, sides.lengths, sides.shapes, chosen.dtype, stream)
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        slopes, *masks = ctx.saved_tensors
        pairs, lengths, shapes, dtype, stream = ctx.args
        lib = _lib.load()
        up = _on(grad.detach().float(), slopes.device)
        grads = [torch.empty(s, dtype=dtype, device=slopes.device) if need else None
                 for s, need in zip(shapes, ctx.needs_input_grad)]
        c, r = (_lib.PreferenceSide(None, None, _ptr(m), n, _ptr(g))
                for m, n, g in zip(masks, lengths, grads))
        args = (c, r, pairs, _FLOATS[dtype], _ptr(slopes), _ptr(up))
        if _on_cpu(stream):
            _lib.check(lib.mlxc_preference_grad_cpu(*args), "preference_loss")
        else:
            run = _Launch(stream, (slopes,))
            with run.uses(slopes, up, *masks, *grads):
                rc = lib.mlxc_preference_grad(*args, run.handle)
            _lib.check(rc, "preference_loss")
            _join_side_stream(stream)
        return (*(None if g is None else g.to(d) for g, d in zip(grads, ctx.devices)), None, None)


def preference_loss(chosen, rejected, ref_chosen=None, ref_rejected=None, *, chosen_mask=None,
                    rejected_mask=None, beta: float = 0.1, label_smoothing: float = 0.0,
                    normalize: bool = False, reduction: str = "mean",
                    return_rewards: bool = False, stream=None):
    """Preference loss of paired log ratios: a float32 scalar.

    With r = the sum of values - reference over a row and z = beta * (r_chosen -
    r_rejected), the mean over the pairs of (1 - label_smoothing) * log(1 +
    e^-z) + label_smoothing * log(1 + e^z).  Values are log-probabilities of
    tokens, or scores of windows: those of one start node differ from
    log-probabilities by the same constant, which the difference drops.

    Args:
        chosen, rejected: [..., T] of one dtype (float32, bfloat16, float16),
            the same pairs and any two lengths T; 1-D: one value a pair.
            window_scores' results go in as they are.  Differentiable.
        ref_chosen, ref_rejected: the same of a reference model (no gradient);
            None: zeros.
        chosen_mask, rejected_mask: bool of the values' shapes, False leaves a
            place out, whatever it holds; None: none left out.  A row with
            nothing left has r = 0.
        normalize: r is the mean over the places left instead of the sum.
        reduction: 'mean' or 'sum' over the pairs (0 of no pairs).
        return_rewards: also return float32 [2, pairs]: beta * r of both sides.
        stream: as in random_walk ('cpu' runs the host twin).
    """
    _check_stream_arg(stream)
    sides = _Sides(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta,
                   label_smoothing, normalize, reduction)
    if _tracked(*sides.values):
        loss, rewards = _PreferenceFunction.apply(*sides.values, sides, stream)
    else:
        loss, rewards, _, _ = _preference(sides, False, False, stream)
    return (loss, rewards) if return_rewards else loss


def preference_loss_grad(chosen, rejected, ref_chosen=None, ref_rejected=None, *, chosen_mask=None,
                         rejected_mask=None, beta: float = 0.1, label_smoothing: float = 0.0,
                         normalize: bool = False, reduction: str = "mean", stream=None):
    """preference_loss with its gradients, in one pass over the values.

    Returns (loss, rewards, d_chosen, d_rejected): the loss, float32 [2, pairs]
    rewards, and its gradients in the values' shapes and dtype (0 in masked
    places).  Arguments as in preference_loss.
    """
    if reduction in ("mean", "sum") and type(label_smoothing) is float and \
            0.0 <= label_smoothing <= 1.0 and _plain(stream, beta, chosen, rejected) and \
            math.isfinite(beta) and all(t is None or isinstance(t, torch.Tensor) for t in
                                        (ref_chosen, ref_rejected, chosen_mask, rejected_mask)):
        res = _fast.preference_loss_grad(
            chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta,
            label_smoothing, (_lib.MLXC_PREFERENCE_NORMALIZE if normalize else 0) |
            (_lib.MLXC_PREFERENCE_SUM if reduction == "sum" else 0))
        if res is not None:
            return res
    _check_stream_arg(stream)
    sides = _Sides(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta,
                   label_smoothing, normalize, reduction)
    loss, rewards, _, grads = _preference(sides, True, False, stream)
    return loss, rewards, grads[0], grads[1]
