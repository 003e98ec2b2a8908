"""The operators that train node embeddings on walks, as they are timed.

A program that trains on this package's walks looks rows of a table up by node
(`embedding`), brings gradients of such rows back to the table
(`embedding_grad`), scores the skip-gram windows of walks (`window_scores`),
brings the scores' gradients back (`window_scores_grad`), and takes a loss of
preferred against other windows or sequences with its gradients
(`preference_loss_grad`).

With `own` false the operators are computed in their plain form, elementary
torch operations in 32 bits, rounded once at the end.

Kinds of case:
  lookup      rows of a table by node, scaled; -1 is no node (a zero row)
  grad        the gradient of a lookup, dense or coalesced: ids ascending and
              their rows, padded with -1 and zero rows to min(nodes, rows)
  scores      the windows of walks: first node against the nodes after it
  scoresgrad  the table's gradient from the scores' gradients
  preference  paired log ratios: loss, rewards and both gradients

Nodes are drawn as an R-MAT graph's degrees are (each bit of a node is set with
probability 0.24), which is how often walks visit them.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # Rows of the start nodes of a Cora-sized graph: launches count.
        {"name": "lookup cora", "kind": "lookup", "rows": 2708, "dim": 64, "dtype": "float32",
         "walks": 2000, "length": 1, "int32": False, "missing": 0.0, "scale": 1.0},
        # Inputs of a sequence model over a batch of 32,768 walks of 80 steps.
        {"name": "lookup walks", "kind": "lookup", "rows": 1 << 20, "dim": 128,
         "dtype": "bfloat16", "walks": 32768, "length": 81, "int32": False, "missing": 0.0,
         "scale": math.sqrt(128)},
        # The gradient of the reference tests' own walks (2,000 of 5 steps).
        {"name": "grad cora", "kind": "grad", "rows": 2708, "dim": 64, "dtype": "float32",
         "walks": 2000, "length": 6, "int32": False, "missing": 0.0, "scale": 1.0,
         "sparse": False},
        # The gradient of "lookup walks": hubs repeat tens of thousands of times.
        {"name": "grad walks", "kind": "grad", "rows": 1 << 20, "dim": 128, "dtype": "bfloat16",
         "walks": 32768, "length": 81, "int32": False, "missing": 0.0, "scale": math.sqrt(128),
         "sparse": False},
        # A mini-batch of edge features of a large graph, coalesced for a sparse
        # optimizer: int32 edge ids, -1 where a walk stayed, an odd row size.
        {"name": "grad edges sparse", "kind": "grad", "rows": 1 << 24, "dim": 100,
         "dtype": "float32", "walks": 1300, "length": 37, "int32": True, "missing": 0.1,
         "scale": 0.1, "sparse": True},
        # One mini-batch of a training loop: 1,300 walks, context 10.
        {"name": "scores batch", "kind": "scores", "rows": 1 << 20, "dim": 128,
         "dtype": "float32", "walks": 1300, "length": 38, "context": 10, "int32": True,
         "scale": 1.0},
        # A large batch: 65,536 walks of 80 steps.
        {"name": "scores large", "kind": "scores", "rows": 1 << 20, "dim": 128,
         "dtype": "bfloat16", "walks": 65536, "length": 81, "context": 10, "int32": False,
         "scale": 1.0},
        # Negative windows, ten nodes each (every window a walk of its own), on a
        # graph of one million nodes that is no power of two, coalesced.
        {"name": "scores grad windows", "kind": "scoresgrad", "rows": 1_000_003, "dim": 100,
         "dtype": "float32", "walks": 37700, "length": 10, "context": 10, "int32": False,
         "scale": 0.1, "sparse": True},
        # The gradient of "scores large".
        {"name": "scores grad large", "kind": "scoresgrad", "rows": 1 << 20, "dim": 128,
         "dtype": "bfloat16", "walks": 65536, "length": 81, "context": 10, "int32": False,
         "scale": 1.0, "sparse": False},
        # The windows of 2,000 short walks against their negatives, no reference.
        {"name": "preference cora", "kind": "preference", "pairs": 2000, "chosen": 5,
         "rejected": 5, "dtype": "float32", "masks": False, "references": False, "beta": 1.0,
         "smoothing": 0.0, "normalize": False},
        # Every window of the large batch against its negative, with the scores of
        # a frozen table as references.
        {"name": "preference windows", "kind": "preference", "pairs": 65536 * 72, "chosen": 9,
         "rejected": 9, "dtype": "float32", "masks": False, "references": True, "beta": 0.5,
         "smoothing": 0.0, "normalize": False},
        # Whole sequences of ragged lengths: 16-bit log-probabilities under masks,
        # some sequences empty, smoothed labels, averaged over the tokens.
        {"name": "preference sequences", "kind": "preference", "pairs": 4097, "chosen": 777,
         "rejected": 1025, "dtype": "bfloat16", "masks": True, "references": True, "beta": 0.1,
         "smoothing": 0.1, "normalize": True},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "grad", "scores", "scoresgrad", "preference"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind == "preference":
        # gradients of a mean over many tokens fall below what float16 holds
        dtype = rng.choice(["float32", "bfloat16"])
        length = _spread(rng, 1, 2000)
        return {"kind": kind, "pairs": _spread(rng, 30, max(60, min(1 << 21, (1 << 24) // length))),
                "chosen": length, "rejected": max(1, int(length * rng.uniform(0.5, 1.2))),
                "dtype": dtype, "masks": rng.random() < 0.5, "references": rng.random() < 0.7,
                "beta": rng.choice([0.05, 0.1, 0.5, 1.0]), "smoothing": rng.choice([0.0, 0.1]),
                "normalize": rng.random() < 0.5}
    dim = rng.choice([16, 33, 50, 64, 96, 100, 128, 200, 256])
    c = {"kind": kind, "rows": _spread(rng, 500, 1 << 21), "dim": dim, "dtype": dtype,
         "int32": rng.random() < 0.4, "scale": rng.choice([1.0, 0.1, math.sqrt(dim)])}
    if kind in ("lookup", "grad"):
        c["length"] = _spread(rng, 1, 100)
        c["walks"] = _spread(rng, 40, max(80, (1 << 28) // (dim * c["length"])))
        c["missing"] = rng.choice([0.0, 0.0, 0.1, 0.9])
    else:
        c["context"] = rng.randint(2, 32)
        c["length"] = c["context"] + (0 if rng.random() < 0.3 else _spread(rng, 1, 100))
        c["walks"] = _spread(rng, 40, max(80, (1 << 27) // (dim * c["length"])))
    if kind in ("grad", "scoresgrad"):
        c["sparse"] = rng.random() < 0.4
    return c


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _nodes(case, g):
    """[walks, length] nodes; a share `missing` of them -1."""
    rows, shape = case["rows"], (case["walks"], case["length"])
    x = torch.zeros(shape, dtype=torch.int64, device="cuda")
    for b in range(max(1, (rows - 1).bit_length())):
        x += (torch.rand(shape, generator=g, device="cuda") < 0.24).long() << b
    x %= rows
    if case.get("missing"):
        x[torch.rand(shape, generator=g, device="cuda") < case["missing"]] = -1
    return x.int() if case["int32"] else x


def prepare(case, seed):
    g = _generator(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "preference":
        pairs = case["pairs"]
        for side, mean in (("chosen", 0.5), ("rejected", -0.5)):
            T = case[side]
            x = rand(pairs, T)
            x += mean
            s["ref_" + side] = (x + 0.1 * rand(pairs, T)).to(dtype) if case["references"] else None
            s[side + "_mask"] = None
            if case["masks"]:
                # a prompt before the answer and padding after it; one in 16 is empty
                first = (torch.rand(pairs, 1, generator=g, device="cuda") * 0.2 * T).long()
                count = (torch.rand(pairs, 1, generator=g, device="cuda") * (T + 1)).long()
                count[torch.rand(pairs, 1, generator=g, device="cuda") < 1 / 16] = 0
                t = torch.arange(T, device="cuda")
                mask = (t >= first) & (t < first + count)
                x = torch.where(mask, x, -math.inf)  # what stands in masked places is no number to use
                s[side + "_mask"] = mask
            s[side] = x.to(dtype)
        return s
    s["nodes"] = _nodes(case, g)
    if kind != "grad":
        s["weight"] = (rand(case["rows"], case["dim"]) / math.sqrt(case["dim"])).to(dtype)
    if kind == "grad":
        s["grad"] = (rand(case["walks"], case["length"], case["dim"]) * 0.01).to(dtype)
    if kind == "scoresgrad":
        C = case["context"]
        s["grad"] = rand(case["walks"], case["length"] - C + 1, C - 1) * 0.01
    return s


# ------------------------------------------------------------- plain forms


def _rows(weight, nodes):
    """Rows of the table in 32 bits, zeros where there is no node."""
    x = nodes.long()
    r = weight[x.clamp(min=0)].float()
    return r.masked_fill((x < 0).unsqueeze(-1), 0.0)


def _plain_grad(rows_grad, nodes, num_rows, sparse, dtype):
    x = nodes.reshape(-1).long()
    g = rows_grad.reshape(x.numel(), -1)
    have = x >= 0
    if sparse:
        # ids ascending, then -1 and zero rows up to the most that there can be
        ids, order = torch.sort(torch.where(have, x, num_rows))
        first = ids < num_rows
        first[1:] &= ids[1:] != ids[:-1]
        at = (torch.cumsum(first.long(), 0) - 1).clamp(min=0)
        cap = min(x.numel(), num_rows)
        ids_out = torch.full((cap,), -1, dtype=torch.int64, device=x.device)
        ids_out[at[first]] = ids[first]
        out = torch.zeros(cap, g.shape[1], dtype=torch.float32, device=g.device)
        out.index_add_(0, at, g[order] * (ids < num_rows).unsqueeze(-1).float())
        return ids_out, out.to(dtype)
    out = torch.zeros(num_rows, g.shape[1], dtype=torch.float32, device=g.device)
    out.index_add_(0, x.clamp(min=0), g * have.unsqueeze(-1).float())
    return out.to(dtype)


def _plain_ratio(x, ref, mask, normalize):
    d = x.float() if ref is None else x.float() - ref.float()
    if mask is not None:
        d = torch.where(mask, d, torch.zeros_like(d))
    r = d.sum(-1)
    n = torch.full_like(r, d.shape[-1]) if mask is None else mask.sum(-1).float()
    share = 1.0 / n.clamp(min=1) if normalize else torch.ones_like(n)
    return r * share, share


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain_preference(s):
    c = s["case"]
    rc, nc = _plain_ratio(s["chosen"], s["ref_chosen"], s["chosen_mask"], c["normalize"])
    rr, nr = _plain_ratio(s["rejected"], s["ref_rejected"], s["rejected_mask"], c["normalize"])
    beta, eps = c["beta"], c["smoothing"]
    z = beta * (rc - rr)
    loss = (1 - eps) * _softplus(-z) + eps * _softplus(z)
    dz = eps / (1 + torch.exp(-z)) - (1 - eps) / (1 + torch.exp(z))
    dz = dz * (beta / c["pairs"])
    grads = []
    for side, d in (("chosen", dz * nc), ("rejected", -dz * nr)):
        x, mask = s[side], s[side + "_mask"]
        g = d.unsqueeze(-1).expand(x.shape)
        grads.append((g.clone() if mask is None else g * mask.float()).to(x.dtype))
    return loss.mean(), torch.stack([beta * rc, beta * rr]), grads[0], grads[1]


def _plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "preference":
        return _plain_preference(s)
    x = s["nodes"]
    if kind == "lookup":
        return (_rows(s["weight"], x) * c["scale"]).to(s["weight"].dtype)
    if kind == "grad":
        return _plain_grad(s["grad"].float() * c["scale"], x, c["rows"], c["sparse"],
                           s["grad"].dtype)
    C = c["context"]
    W = c["length"] - C + 1
    u = _rows(s["weight"], x)
    if kind == "scores":
        return torch.stack([(u[:, :W] * u[:, k:k + W]).sum(-1) for k in range(1, C)],
                           dim=-1) * c["scale"]
    du = torch.zeros_like(u)
    for k in range(1, C):
        d = s["grad"][:, :, k - 1].unsqueeze(-1) * c["scale"]
        du[:, :W] += d * u[:, k:k + W]
        du[:, k:k + W] += d * u[:, :W]
    return _plain_grad(du, x, c["rows"], c["sparse"], s["weight"].dtype)


# ------------------------------------------------------------- the passes


def run(state):
    if not own:
        return _plain(state)
    import mlx_cluster_amd as mc
    c = state["case"]
    kind = c["kind"]
    if kind == "preference":
        return mc.preference_loss_grad(
            state["chosen"], state["rejected"], state["ref_chosen"], state["ref_rejected"],
            chosen_mask=state["chosen_mask"], rejected_mask=state["rejected_mask"],
            beta=c["beta"], label_smoothing=c["smoothing"], normalize=c["normalize"])
    # the nodes come from a walk call, which has checked them
    if kind == "lookup":
        return mc.embedding(state["weight"], state["nodes"], scale=c["scale"], check=False)
    if kind == "grad":
        return mc.embedding_grad(state["grad"], state["nodes"], c["rows"], scale=c["scale"],
                                 sparse=c["sparse"], check=False)
    if kind == "scores":
        return mc.window_scores(state["weight"], state["nodes"], c["context"], scale=c["scale"],
                                check=False)
    return mc.window_scores_grad(state["grad"], state["weight"], state["nodes"], c["context"],
                                 scale=c["scale"], sparse=c["sparse"], check=False)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    kind = case["kind"]
    if kind == "preference":
        values = case["pairs"] * (case["chosen"] + case["rejected"])
        per = size * (3 if case["references"] else 2) + (1 if case["masks"] else 0)
        return {"bytes": values * per + 8 * case["pairs"] + 4,
                "flops": values * (2 if case["references"] else 1) + 20 * case["pairs"]}
    T, D, V = case["walks"] * case["length"], case["dim"], case["rows"]
    ids = T * (4 if case["int32"] else 8)
    row = D * size
    touched = min(V, T)  # rows of the table that the call can reach
    if kind == "lookup":
        return {"bytes": ids + (touched + T) * row, "flops": T * D}
    if kind == "grad":
        out = touched * (row + 8) if case["sparse"] else V * row
        return {"bytes": ids + T * row + out, "flops": 2 * T * D}
    C = case["context"]
    pairs = case["walks"] * (case["length"] - C + 1) * (C - 1)
    if kind == "scores":
        return {"bytes": ids + touched * row + 4 * pairs, "flops": 2 * pairs * D}
    out = touched * (row + 8) if case["sparse"] else V * row
    return {"bytes": ids + touched * row + 4 * pairs + out, "flops": 4 * pairs * D + T * D}


# ------------------------------------------------------------- in 64 bits


def _exact_scatter(ids, values, num_rows, sparse):
    """values [T, D] (float64) added up by id; ids of -1 are left out."""
    cap = min(ids.numel(), num_rows)
    keep = ids >= 0
    ids, values = ids[keep], values[keep]
    if sparse:
        ids_out, ids = torch.unique(ids, sorted=True, return_inverse=True)
        num_rows = cap
    out = torch.zeros(num_rows, values.shape[1], dtype=torch.float64, device=values.device)
    out.scatter_add_(0, ids.unsqueeze(1).expand(-1, values.shape[1]), values)
    if not sparse:
        return out
    return torch.nn.functional.pad(ids_out, (0, cap - ids_out.numel()), value=-1), out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "preference":
        ratio, share, beta = {}, {}, case["beta"]
        for side in ("chosen", "rejected"):
            d = s[side].double()
            if s["ref_" + side] is not None:
                d -= s["ref_" + side].double()
            n = torch.full((case["pairs"],), float(case[side]), dtype=torch.float64, device="cuda")
            if s[side + "_mask"] is not None:
                d.masked_fill_(~s[side + "_mask"], 0.0)
                n = s[side + "_mask"].double().sum(1)
            share[side] = 1 / n.clamp(min=1) if case["normalize"] else torch.ones_like(n)
            ratio[side] = d.sum(1) * share[side]
        z = beta * (ratio["chosen"] - ratio["rejected"])
        eps, zero = case["smoothing"], torch.zeros_like(z)
        loss = (1 - eps) * torch.logaddexp(zero, -z) + eps * torch.logaddexp(zero, z)
        slope = (torch.sigmoid(z) - (1 - eps)) * beta / case["pairs"]
        grads = []
        for side, sign in (("chosen", 1.0), ("rejected", -1.0)):
            g = (sign * slope * share[side]).unsqueeze(1).repeat(1, case[side])
            if s[side + "_mask"] is not None:
                g.masked_fill_(~s[side + "_mask"], 0.0)
            grads.append(g)
        return (loss.sum() / case["pairs"], beta * torch.stack([ratio["chosen"], ratio["rejected"]]),
                grads[0], grads[1])
    nodes = s["nodes"].long()
    if kind == "grad":
        return _exact_scatter(nodes.reshape(-1),
                              s["grad"].double().reshape(nodes.numel(), -1) * case["scale"],
                              case["rows"], case["sparse"])
    table = torch.cat([s["weight"].double(), s["weight"].new_zeros(1, case["dim"]).double()])
    if kind == "lookup":
        return table[nodes] * case["scale"]
    # the scores are diagonals of every walk's product of rows, 64-bit matrices;
    # their gradient is that band, mirrored, times the rows
    C, M = case["context"], case["length"]
    W = M - C + 1
    j = torch.arange(W, device="cuda").unsqueeze(1)
    k = torch.arange(1, C, device="cuda").unsqueeze(0)
    at = (j * M + j + k).reshape(-1)
    step = max(1, (1 << 26) // (M * max(M, case["dim"])))
    parts = []
    for i in range(0, case["walks"], step):
        u = table[nodes[i:i + step]]
        if kind == "scores":
            p = torch.matmul(u, u.transpose(1, 2).contiguous()).reshape(-1, M * M)
            parts.append(p[:, at].reshape(-1, W, C - 1) * case["scale"])
        else:
            b = torch.zeros(u.shape[0], M * M, dtype=torch.float64, device="cuda")
            b[:, at] = s["grad"][i:i + step].double().reshape(u.shape[0], -1) * case["scale"]
            b = b.reshape(-1, M, M)
            parts.append(torch.matmul((b + b.transpose(1, 2)).contiguous(), u))
    if kind == "scores":
        return torch.cat(parts)
    return _exact_scatter(nodes.reshape(-1), torch.cat(parts).reshape(nodes.numel(), -1),
                          case["rows"], case["sparse"])
