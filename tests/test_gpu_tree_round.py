"""Accepted paths moved in the pools, and a whole draft-tree round."""

import math

import pytest
import torch

from tests.tree_cases import FP8, make_case, pack_bits, reference
from tests.tree_rounds import greedy_tree, random_trees, sampled_inputs

pytestmark = pytest.mark.gpu


def moved(pool, tables, starts, path, accepted, bs):
    """The moves one by one on a copy, a source read when its turn comes."""
    out = pool.clone()
    t3 = tables if tables.ndim == 3 else tables[:, None]
    for r in range(path.shape[0]):
        for plane in range(t3.shape[1]):
            tb = t3[r, plane]
            for j in range(1, min(max(int(accepted[r]), 0), path.shape[1] - 1) + 1):
                node = int(path[r, j])
                src, dst = int(starts[r]) + node, int(starts[r]) + j
                if node <= j or src // bs >= len(tb) or dst // bs >= len(tb):
                    continue
                sb, db = int(tb[src // bs]), int(tb[dst // bs])
                if 0 <= sb < pool.shape[0] and 0 <= db < pool.shape[0]:
                    out[db, :, dst % bs] = out[sb, :, src % bs]
    return out


def paths(n, w, g):
    path = torch.full((n, w + 1), -1, dtype=torch.int64)
    accepted = torch.randint(0, w + 1, (n,), generator=g)
    accepted[0] = w
    for r in range(n):
        a = int(accepted[r])
        path[r, 0] = 0
        path[r, 1:a + 1] = (torch.randperm(w, generator=g)[:a] + 1).sort().values
    return path, accepted


@pytest.mark.parametrize("n,w,layers,tail,dtype,bs,planes", [
    (1, 1, 1, (1, 64), torch.bfloat16, 16, 0),
    (5, 16, 3, (4, 128), torch.bfloat16, 16, 0),
    (3, 40, 2, (2, 96), FP8, 16, 0),
    (4, 9, 2, (3, 7), torch.bfloat16, 8, 0),       # 42 bytes a token: byte moves
    (4, 9, 2, (3,), torch.float32, 16, 0),         # an fp8 cache's scale pool
    (2, 255, 1, (1, 64), torch.float16, 16, 0),
    (3, 12, 2, (2, 64), torch.float32, 5, 3),      # planes, odd blocks
    (2, 12, 1, (40, 256), torch.bfloat16, 16, 2),  # 20 KB a token
])
def test_commit_moves_the_path(pkg, dev, n, w, layers, tail, dtype, bs, planes):
    g = torch.Generator().manual_seed(n + w)
    width = (3 * bs + w) // bs + 1
    count = n * max(planes, 1) * width
    k, v = ((torch.randn(count + 2, layers, bs, *tail, generator=g) * 9).to(dtype) for _ in range(2))
    tables = torch.randperm(count, generator=g).int().view(n, *([planes] if planes else []), width)
    starts = torch.randint(0, 3 * bs, (n,), generator=g)
    path, accepted = paths(n, w, g)
    kd, vd = k.to(dev), v.to(dev)
    pkg.commit_tree_kv(kd, vd, tables.to(dev), starts.to(dev), path.to(dev), accepted.to(dev), bs)
    bits = lambda x: x.view(torch.uint8) if x.dtype == FP8 else x  # noqa: E731
    for got, old in ((kd, k), (vd, v)):
        want = moved(bits(old), tables, starts, path, accepted, bs)
        assert torch.equal(bits(got).cpu(), want)


def test_commit_leaves_what_it_cannot_place(pkg, dev):
    """Positions past the table, blocks outside the pool, counts past the path, paths that do
    not ascend: nothing outside the listed moves changes."""
    g = torch.Generator().manual_seed(1)
    k = torch.randn(20, 2, 4, 2, 16, generator=g)
    tables = torch.tensor([[1, 2, 3], [4, -1, 5], [6, 99, 7], [8, 9, 10], [11, 12, 13]],
                          dtype=torch.int32)
    starts = torch.tensor([6, 2, 2, -3, 1])
    path = torch.tensor([[0, 2, 3, 5, 6], [0, 1, 2, 3, 5], [0, 3, 4, 5, 7], [0, 2, 3, 4, 5],
                         [0, 1, 1, 300, 9]])
    accepted = torch.tensor([99, 4, 4, 4, 4])
    kd, vd = k.to(dev), (-k).to(dev)
    pkg.commit_tree_kv(kd, vd, *to_dev(dev, tables, starts, path, accepted), 4)
    want = moved(k, tables, torch.where(starts < 0, 1000, starts), path, accepted, 4)
    assert torch.equal(kd.cpu(), want) and torch.equal(vd.cpu(), -want)


def test_commit_of_far_positions(pkg, dev):
    """Starts that no table reaches, up to the largest integer: nothing moves."""
    g = torch.Generator().manual_seed(4)
    k = torch.randn(6, 2, 4, 2, 16, generator=g)
    tables = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32)
    starts = torch.tensor([(1 << 63) - 1, (1 << 63) - 3, 8])
    path, accepted = torch.tensor([[0, 3, 5, 6]] * 3), torch.full((3,), 3)
    kd, vd = k.to(dev), (-k).to(dev)
    pkg.commit_tree_kv(kd, vd, *to_dev(dev, tables, starts, path, accepted), 4)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), -k)


def to_dev(dev, *xs):
    return [x.to(dev) for x in xs]


def test_commit_strided_pools(pkg, dev):
    """Layers of a larger allocation."""
    g = torch.Generator().manual_seed(2)
    big = torch.randn(10, 7, 16, 2, 64, generator=g).bfloat16()
    path, accepted = paths(2, 10, g)
    tables = torch.arange(10).view(2, 5).int()
    starts = torch.tensor([5, 40])
    kd, vd = big.to(dev), big.flip(0).contiguous().to(dev)
    pkg.commit_tree_kv(kd[:, 2:5], vd[:, 2:5], *to_dev(dev, tables, starts, path, accepted), 16)
    want = big.clone()
    want[:, 2:5] = moved(big[:, 2:5], tables, starts, path, accepted, 16)
    assert torch.equal(kd.cpu(), want)


@pytest.mark.parametrize("kv", ["same", "fp8_vector"])
def test_a_whole_round(pkg, dev, kv):
    """Masks, attention, greedy acceptance, commit and log probabilities of three requests; the
    chain left in the cache then attends like the path did."""
    nodes, ctx, w = [9, 5, 12], [70, 33, 140], 11
    c = make_case(nodes, ctx, 4, 2, 64, torch.bfloat16, kv, seed=40)
    g = torch.Generator().manual_seed(41)
    parents = random_trees(3, w, g)
    for s, m in enumerate(nodes):
        parents[s, :m - 1] = torch.tensor(c.parents[s])
    cu, pd = c.cu.to(dev), parents.to(dev)
    mask = pkg.tree_masks(pd, cu, int(c.cu[-1]))
    assert torch.equal(mask.cpu(), c.mask)
    # pools whole, so that the commit sees every layer (two: the second attends)
    backend = pkg.create_backend("auto", dev, torch.bfloat16, 64, c.block)
    base = lambda x: x._base if x is not None and x._base is not None else x  # noqa: E731
    kp, vp = base(c.k).to(dev), base(c.v).to(dev)
    scales = (None, None)
    if kv != "same":
        ksp, vsp = base(c.k_scale).to(dev), base(c.v_scale).to(dev)
        scales = (ksp[:, 1], vsp[:, 1])
    q, tables = c.q.to(dev), c.tables.to(dev)
    out = backend.tree(q, kp[:, 1], vp[:, 1], tables, c.lengths.to(dev), cu, max(nodes), mask, *scales)
    want, tol = reference(c)
    assert ((out.double().cpu() - want).abs() <= tol).all()
    # logits of a linear head over the attention output, padded to [n, W + 1, V]
    vocab = 500
    head = torch.randn(256, vocab, generator=g).to(dev)
    rows = (out.float().flatten(1) @ head).cpu()
    logits = torch.randn(3, w + 1, vocab, generator=g)
    for s, m in enumerate(nodes):
        logits[s, :m] = rows[int(c.cu[s]):int(c.cu[s]) + m]
    drafts = torch.tensor([m - 1 for m in nodes])
    best = logits.argmax(-1)
    tokens = best.gather(1, parents)
    tokens[:, 1::3] = 3  # some drafts are wrong
    got = pkg.greedy_tree_accept(*to_dev(dev, tokens, parents, drafts, logits))
    want_g = greedy_tree(tokens, parents, drafts, logits)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want_g))
    targets, path, accepted, _ = got
    assert accepted.max() >= 2
    # log probabilities of the emitted tokens at the nodes that decided them
    flat = torch.where(path >= 0, path + (w + 1) * torch.arange(3, device=dev)[:, None], path).flatten()
    emitted = targets.flatten().gather(0, flat.clamp(min=0))
    lp = pkg.token_logprobs(logits.flatten(0, 1).to(dev), emitted, rows=flat, top_n=2)
    live = (flat >= 0).cpu()
    assert (lp.rank.cpu()[live] == 1).all() and (lp.rank.cpu()[~live] == 0).all()
    ref = torch.log_softmax(logits.flatten(0, 1).double(), -1)[flat.cpu()[live], emitted.cpu()[live]]
    assert (lp.logprob.double().cpu()[live] - ref).abs().max() <= 1e-5
    # the path's keys and values behind the prefix
    starts = (c.lengths - torch.tensor(nodes)).long().to(dev)
    pkg.commit_tree_kv(kp, vp, tables, starts, path, accepted, c.block)
    if kv != "same":
        pkg.commit_tree_kv(ksp, vsp, tables, starts, path, accepted, c.block)
    # the accepted nodes' rows, now a chain: each sees what it saw
    keep = [int(c.cu[s]) + int(i) for s in range(3) for i in path[s, :int(accepted[s]) + 1]]
    counts = [int(a) + 1 for a in accepted]
    ccu = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
    lens = (starts.cpu() + torch.tensor(counts)).int()
    chain_mask = pack_bits([(2 << i) - 1 for m in counts for i in range(m)], 1)
    again = backend.tree(q[keep], kp[:, 1], vp[:, 1], tables, lens.to(dev), ccu.to(dev), max(counts),
                         chain_mask.to(dev), *scales)
    assert ((again.double() - out[keep].double()).cpu().abs() <= 2 * tol[keep]).all()
    causal = backend.prefill(q[keep], kp[:, 1], vp[:, 1], tables, lens.to(dev), ccu.to(dev),
                             max(counts), *scales)
    assert ((causal.double() - out[keep].double()).cpu().abs() <= 2 * tol[keep]).all()
    assert math.isfinite(float(again.float().sum()))


def test_operators_keep_their_schemas(pkg, dev):
    """torch.library.opcheck's schema and fake-tensor checks of every operator of the round."""
    checks = ("test_schema", "test_faketensor")
    ops = torch.ops.rlt_mi355x
    c = make_case([9, 5], [70, 33], 4, 2, 64, torch.bfloat16, seed=50)
    a = to_dev(dev, *sampled_inputs(3, 5, 300, seed=1))
    path, accepted = paths(2, 10, torch.Generator().manual_seed(2))
    pool = torch.randn(10, 2, 16, 2, 64, device=dev)
    tables = torch.arange(10).view(2, 5).int()
    for op, args in (
            (ops.tree_attention, (*to_dev(dev, c.q, c.k, c.v, c.tables, c.lengths, c.cu), 9,
                                  c.mask.to(dev))),
            (ops.tree_masks, (a[1], torch.tensor([0, 6, 9, 12], dtype=torch.int32, device=dev), 12)),
            (ops.tree_accept, a),
            (ops.greedy_tree_accept, (*a[:3], a[4])),
            (ops.token_logprobs, (a[4][0], torch.zeros(6, dtype=torch.int64, device=dev), None, 3)),
            (ops.commit_tree_kv, (pool, pool.clone(), *to_dev(dev, tables, torch.tensor([5, 40]), path,
                                                              accepted), 16))):
        torch.library.opcheck(op, tuple(args), test_utils=checks)
