"""Plain float64 forms of the draft-tree round's decisions, request by request."""

import math

import numpy as np
import torch

from tests.tree_cases import random_parents


def tree_accept(tokens, parents, drafts, q, p, u_accept, u_final):
    """The definition, with the weights left at a node kept explicitly."""
    n, w = tokens.shape
    vocab = p.shape[-1]
    path = torch.full((n, w + 1), -1, dtype=torch.int64)
    out = torch.zeros((n, w + 1), dtype=torch.int64)
    accepted = torch.zeros(n, dtype=torch.int64)
    final = torch.zeros(n, dtype=torch.int64)
    error = torch.zeros(n, dtype=torch.bool)
    for r in range(n):
        live = min(max(int(drafts[r]), 0), w)
        bad = live != int(drafts[r])
        node, count, mass = 0, 0, 1.0
        y = p[r, 0].double()
        path[r, 0] = 0
        for j in range(live):
            if bad:
                break
            if int(parents[r, j]) != node:
                continue
            t = int(tokens[r, j])
            if not 0 <= t < vocab:
                bad = True
                break
            qt, pt = float(q[r, node, t]), float(p[r, node, t])
            if not (qt > 0 and math.isfinite(qt) and math.isfinite(pt)):
                bad = True
                break
            if float(u_accept[r, j]) * mass * qt < float(y[t]):
                out[r, count] = t
                count += 1
                node, mass = j + 1, 1.0
                y = p[r, node].double()
                path[r, count] = node
            else:
                y = (y - mass * q[r, node].double()).clamp_min(0)
                mass = float(y.sum())
                bad = not (math.isfinite(mass) and mass > 0)
        if not bad:
            y = y.clamp_min(0)
            cdf = y.cumsum(0)
            total = float(cdf[-1])
            bad = not (math.isfinite(total) and total > 0)
        if not bad:
            at = min(float(u_final[r]) * total, float(np.nextafter(total, 0.0)))
            final[r] = min(int((cdf <= at).sum()), vocab - 1)
        out[r, count] = final[r]
        accepted[r] = count
        error[r] = bad
    return path, out, accepted, final, error


def greedy_tree(tokens, parents, drafts, logits):
    n, w = tokens.shape
    x = logits.double()
    best = x.nan_to_num(math.inf, math.inf, -math.inf) if not torch.isnan(x).any() else None
    if best is None:
        # NaN comes first
        best = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)
        best = torch.where(torch.isnan(x).any(-1, keepdim=True) & ~torch.isnan(x),
                           torch.full_like(x, -math.inf), best)
    top = best.amax(-1, keepdim=True)
    columns = torch.arange(x.shape[-1])
    targets = torch.where(best == top, columns, x.shape[-1]).amin(-1)
    path = torch.full((n, w + 1), -1, dtype=torch.int64)
    accepted, last = [], []
    for r in range(n):
        live = min(max(int(drafts[r]), 0), w)
        node, count = 0, 0
        path[r, 0] = 0
        while True:
            hits = [j for j in range(node, live)
                    if int(parents[r, j]) == node and int(tokens[r, j]) == int(targets[r, node])]
            if not hits:
                break
            node = hits[0] + 1
            count += 1
            path[r, count] = node
        accepted.append(count)
        last.append(int(targets[r, node]))
    return targets, path, torch.tensor(accepted), torch.tensor(last)


def random_trees(n, w, g):
    return torch.tensor([random_parents(w, g) if w else [] for _ in range(n)],
                        dtype=torch.int64).view(n, w)


def sampled_inputs(n, w, vocab, seed, sharp=3.0, noise=1.0):
    """p, q and drafts drawn from q at their parents."""
    g = torch.Generator().manual_seed(seed)
    draft = torch.randn(n, max(w, 1), vocab, generator=g) * sharp
    target = torch.cat([draft[:, :w], draft[:, :1].flip(-1)], 1)
    target = target + torch.randn(n, w + 1, vocab, generator=g) * noise
    q, p = draft[:, :w].softmax(-1).contiguous(), target.softmax(-1)
    parents = random_trees(n, w, g)
    tokens = torch.zeros(n, w, dtype=torch.int64)
    for j in range(w):
        rows = q[torch.arange(n), parents[:, j]]
        tokens[:, j] = torch.multinomial(rows, 1, generator=g)[:, 0]
    drafts = torch.randint(0, w + 1, (n,), generator=g)
    drafts[0] = w
    return (tokens, parents, drafts, q, p, torch.rand(n, w, generator=g),
            torch.rand(n, generator=g))
