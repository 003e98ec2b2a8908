"""Node embeddings trained on random walks, from the edge list to node classes.

A graph of communities is walked; the windows of the walks are preferred to
windows of random nodes (`window_scores`, `preference_loss_grad`, and the way
back, `window_scores_grad`); on the way a few labelled nodes pull their rows
towards their class (`embedding`, and its coalesced gradient,
`embedding_grad(sparse=True)`).  Then every other node is classified by its row.

    python examples/train_embeddings.py               # on the GPU
    python examples/train_embeddings.py --device cpu  # host twins
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import mlx_cluster_amd as mlx_cluster  # noqa: E402


def community_graph(nodes: int, classes: int, degree: int, generator) -> tuple:
    """Edges of a graph whose nodes have four of five neighbours in their own class."""
    label = torch.randint(0, classes, (nodes,), generator=generator)
    order = torch.argsort(label)
    first = torch.searchsorted(label[order], torch.arange(classes))
    size = torch.bincount(label, minlength=classes)
    row = torch.arange(nodes).repeat_interleave(degree)
    own = label[row]
    inside = order[first[own] + (torch.rand(row.numel(), generator=generator) * size[own]).long()]
    outside = torch.randint(0, nodes, (row.numel(),), generator=generator)
    col = torch.where(torch.rand(row.numel(), generator=generator) < 0.8, inside, outside)
    return torch.stack([row, col]), label


def train(nodes=3000, classes=5, dim=32, steps=60, batch=1500, walk_length=12, context=5, rate=20.0,
          labelled=0.02, device="cuda", seed=0, log=print):
    """Returns (first losses, last losses, share of unlabelled nodes classified right)."""
    generator = torch.Generator().manual_seed(seed)
    stream = "cpu" if device == "cpu" else None
    edges, label = community_graph(nodes, classes, 8, generator)
    rowptr, col = mlx_cluster.to_csr(edges.to(device), nodes, symmetrize=True, dedup=True)
    weight = (torch.randn(nodes, dim, generator=generator) / dim**0.5).to(device)
    label = label.to(device)
    known = (torch.rand(nodes, generator=generator) < labelled).nonzero().flatten().to(device)
    centres = torch.randn(classes, dim, generator=generator).to(device)
    losses = []
    for step in range(steps):
        start = torch.randint(0, nodes, (batch,), generator=generator).to(device)
        walks = mlx_cluster.rejection_sampling(rowptr, col, start, walk_length, 1.0, 0.5,
                                               seed=seed + step, rule="node2vec", stream=stream)
        windows = walk_length + 2 - context
        other = mlx_cluster.negative_windows(start, walk_length, context, nodes, seed=seed + step,
                                             stream=stream)
        # negative windows come window by window: walk n's j-th is row j * batch + n
        other = other.reshape(windows, batch, context).transpose(0, 1).reshape(-1, context)

        # windows of the walks against windows of random nodes
        chosen = mlx_cluster.window_scores(weight, walks, context, check=False, stream=stream)
        rejected = mlx_cluster.window_scores(weight, other, check=False, stream=stream)
        loss, _, d_chosen, d_rejected = mlx_cluster.preference_loss_grad(
            chosen, rejected.reshape(chosen.shape), beta=0.5, normalize=True, stream=stream)
        grad = mlx_cluster.window_scores_grad(d_chosen, weight, walks, context, check=False,
                                              stream=stream)
        grad += mlx_cluster.window_scores_grad(d_rejected.reshape(rejected.shape), weight, other,
                                               check=False, stream=stream)
        weight -= rate * nodes**0.5 * grad

        # labelled nodes towards their class: the rows by node, and only theirs back
        rows = mlx_cluster.embedding(weight, known, check=False, stream=stream)
        p = torch.softmax(rows @ centres.t(), dim=1)
        p[torch.arange(known.numel(), device=rows.device), label[known]] -= 1.0
        ids, pull = mlx_cluster.embedding_grad((p @ centres) / known.numel(), known, nodes,
                                               sparse=True, check=False, stream=stream)
        have = ids >= 0
        weight[ids[have]] -= rate * pull[have]
        losses.append(float(loss))
        if step % 20 == 0 or step == steps - 1:
            log(f"step {step}: loss {losses[-1]:.4f}")

    # a node's class: the one whose labelled nodes' rows lie nearest on average
    unit = torch.nn.functional.normalize(mlx_cluster.embedding(
        weight, torch.arange(nodes, device=device), scale=dim**0.5, stream=stream), dim=1)
    near = unit @ unit[known].t()
    score = torch.stack([near[:, label[known] == c].mean(dim=1) if bool((label[known] == c).any())
                         else torch.full((nodes,), -1.0, device=device) for c in range(classes)], 1)
    rest = torch.ones(nodes, dtype=torch.bool, device=device)
    rest[known] = False
    right = float((score.argmax(1) == label)[rest].float().mean())
    log(f"{100 * right:.1f}% of the unlabelled nodes classified right ({classes} classes)")
    return losses[:3], losses[-3:], right


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--device", default="cuda", choices=["cuda", "cpu"])
    parser.add_argument("--nodes", type=int, default=3000)
    parser.add_argument("--steps", type=int, default=60)
    args = parser.parse_args()
    train(nodes=args.nodes, steps=args.steps, device=args.device)
