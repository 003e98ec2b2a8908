"""The training operators in 64 bits, plainly, with the rounding that float32
sums may add: every function returns (value, bound), tensors of float64, and an
implementation that adds in float32 in any order and rounds once to `dtype` lies
within bound of value.

A sum of n terms t in float32, each a product or difference that is rounded
once itself, is off by at most (n + 2) * 2^-24 * sum |t| to first order, in any
order of adding; rounding the result to a type of p bits adds 2^-p of its size,
or half of its smallest subnormal.
"""
import torch

U32 = 2.0**-24
ROUND = {torch.float32: (2.0**-24, 2.0**-150), torch.bfloat16: (2.0**-8, 2.0**-134),
         torch.float16: (2.0**-11, 2.0**-25)}


def stored(value, sums_bound, dtype):
    u, least = ROUND[dtype]
    return value, 1.01 * (sums_bound + u * (value.abs() + sums_bound) + least)


def rows_of(weight, nodes):
    x = nodes.long()
    w = weight.double()
    valid = (x >= 0) & (x < w.shape[0])
    r = w[torch.where(valid, x, 0)] if w.shape[0] else torch.zeros(*x.shape, w.shape[1]).double()
    return torch.where(valid.unsqueeze(-1), r, 0.0), valid


def embedding(weight, nodes, scale):
    r, _ = rows_of(weight, nodes)
    v = r * scale
    return stored(v, 2 * U32 * v.abs(), weight.dtype)  # the factor's own rounding, the product's


def _coalesced(values, sizes, counts, nodes, num_rows, scale, dtype, sparse):
    """values, sizes [T, D] by place: terms and the sums of their terms' absolute values;
    counts [T]: how many terms each is a sum of."""
    D = values.shape[1]
    x = nodes.reshape(-1).long()
    total = torch.zeros(num_rows, D, dtype=torch.float64)
    size, n = torch.zeros_like(total), torch.zeros(num_rows, 1, dtype=torch.float64)
    for i, v in enumerate(x.tolist()):
        if 0 <= v < num_rows:
            total[v] += values[i]
            size[v] += sizes[i]
            n[v] += counts[i]
    value, bound = stored(total * scale, (n + 4) * U32 * size * abs(scale), dtype)
    if not sparse:
        return value, bound
    ids = sorted({v for v in x.tolist() if 0 <= v < num_rows})
    cap = min(x.numel(), num_rows)
    pad = cap - len(ids)
    at = torch.tensor(ids, dtype=torch.int64)
    zero = torch.zeros(pad, D, dtype=torch.float64)
    return (torch.cat([at, torch.full((pad,), -1)]), torch.cat([value[at], zero]),
            torch.cat([bound[at], zero]))


def embedding_grad(grad, nodes, num_rows, scale, dtype, sparse=False):
    g = grad.double().reshape(nodes.numel(), grad.shape[-1])
    return _coalesced(g, g.abs(), torch.ones(g.shape[0], 1).double(), nodes, num_rows, scale, dtype,
                      sparse)


def window_scores(weight, walks, C, scale):
    r, valid = rows_of(weight, walks)
    N, M = walks.shape
    W, D = M - C + 1, r.shape[-1]
    out = torch.zeros(N, W, C - 1, dtype=torch.float64)
    size = torch.zeros_like(out)
    for j in range(W):
        for k in range(1, C):
            out[:, j, k - 1] = (r[:, j] * r[:, j + k]).sum(-1)
            size[:, j, k - 1] = (r[:, j] * r[:, j + k]).abs().sum(-1)
    return stored(out * scale, (D + 4) * U32 * size * abs(scale), torch.float32)


def window_scores_grad(grad, weight, walks, C, scale, dtype, sparse=False):
    r, valid = rows_of(weight, walks)
    N, M = walks.shape
    W, D = M - C + 1, r.shape[-1]
    du = torch.zeros(N, M, D, dtype=torch.float64)
    size = torch.zeros_like(du)
    n = torch.zeros(N, M, 1, dtype=torch.float64)
    for j in range(W):
        for k in range(1, C):
            both = (valid[:, j] & valid[:, j + k]).unsqueeze(-1)
            g = torch.where(both, grad[:, j, k - 1].double().unsqueeze(-1), 0.0)
            for a, b in ((j, j + k), (j + k, j)):
                du[:, a] += g * r[:, b]
                size[:, a] += (g * r[:, b]).abs()
                n[:, a] += 1
    return _coalesced(du.reshape(-1, D), size.reshape(-1, D), n.reshape(-1, 1), walks,
                      weight.shape[0], scale, dtype, sparse)


def preference(sides, beta, smoothing=0.0, normalize=False, total=False):
    """sides: two of (values, reference or None, mask or None), [B, T].  Returns
    loss, rewards and the gradients, each (value, bound)."""
    r, rb, share = [], [], []
    for values, ref, mask in sides:
        v = values.double()
        f = torch.zeros_like(v) if ref is None else ref.double()
        m = torch.ones_like(v, dtype=torch.bool) if mask is None else mask.bool()
        d = torch.where(m, v - f, 0.0)
        n = m.sum(-1).double()
        s = 1 / n.clamp(min=1) if normalize else torch.ones_like(n)
        r.append(beta * d.sum(-1) * s)
        rb.append((n + 6) * U32 * abs(beta) * d.abs().sum(-1) * s)
        share.append((s, m))
    z, zb = r[0] - r[1], rb[0] + rb[1]
    zb = zb + U32 * z.abs()
    B = max(1, z.numel())
    soft = lambda x: torch.nn.functional.softplus(x, threshold=1e9)
    zero = torch.zeros_like(z)
    loss = ((1 - smoothing) * soft(-z) if smoothing < 1 else zero) + \
        (smoothing * soft(z) if smoothing > 0 else zero)
    slope = ((smoothing - 1) * torch.sigmoid(-z) if smoothing < 1 else zero) + \
        (smoothing * torch.sigmoid(z) if smoothing > 0 else zero)
    # softplus has a slope of at most 1, sigma one of at most 1/4; expf, log1pf
    # and the divisions take a few units in the last place each
    lb = zb + 16 * U32 * (loss + 1)
    scale = 1.0 if total else 1.0 / B
    loss_out = (loss.sum() * scale, (lb.sum() + (B + 4) * U32 * loss.sum()) * scale)
    grads = []
    for sign, (s, m) in ((1, share[0]), (-1, share[1])):
        g = sign * slope * beta * scale * s
        # an exponent off by zb moves sigma by at most zb of its own size
        gb = (zb * slope.abs() + 16 * U32 * slope.abs() + U32 * 4) * abs(beta) * scale * s
        g = torch.where(m, g.unsqueeze(-1), 0.0)
        gb = torch.where(m, gb.unsqueeze(-1), 0.0)
        grads.append(stored(g, gb, sides[0][0].dtype))
    rewards = (torch.stack(r), torch.stack(rb) + U32 * torch.stack(r).abs())
    return loss_out, rewards, grads[0], grads[1]


def close(got, value, bound):
    """got within bound of value; infinities and NaN where value has them."""
    got, value = got.detach().cpu().double(), value.double()
    assert got.shape == value.shape, (got.shape, value.shape)
    odd = ~torch.isfinite(value)
    same = torch.where(torch.isnan(value), torch.isnan(got), got == value)
    assert bool(same[odd].all()), "other infinities or NaN"
    off = ((got - value).abs() - bound)[~odd]
    assert off.numel() == 0 or float(off.max()) <= 0, f"off by {float(off.max())} over the bound"


# Rows of a walk, in the ways that go wrong: (num_walks, nodes, context).
WINDOWS = [(1, 2, 2), (3, 5, 5), (2, 16, 2), (5, 17, 10), (4, 33, 32), (3, 40, 17), (7, 81, 10),
           (130, 10, 10), (2, 100, 32)]
DIMS = [1, 2, 7, 16, 33, 64, 100, 128, 200, 260]


def make_nodes(g, shape, num_rows, missing=0.0, hub=0.0):
    """Nodes in [0, num_rows), a share `missing` of them -1 and `hub` of them 1 (or 0)."""
    x = torch.randint(0, max(1, num_rows), shape, generator=g)
    x[torch.rand(shape, generator=g) < hub] = min(1, num_rows - 1)
    x[torch.rand(shape, generator=g) < missing] = -1
    if num_rows == 0:
        x.fill_(-1)
    return x
