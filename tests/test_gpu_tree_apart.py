"""Tree attention of large batches: the kv groups of a workgroup take neighbouring heads apart."""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_tree_edges import attend
from tests.tree_cases import FP8, Case, ancestor_bits, pack_bits, random_parents
from tests.tree_dense import dense, sees

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
BLOCK, SHARED = 16, 48


def make_batch(nodes, ctx, hq, hkv, dim, dtype, kv, seed):
    """``tree_cases.make_case`` for many long sequences: prefixes lie in a few blocks that all
    share, the blocks that hold a tree are its own.  What no sequence owns is NaN."""
    g = torch.Generator().manual_seed(seed)
    c = Case()
    c.nodes, c.ctx, c.block = nodes, ctx, BLOCK
    width = max(1, max(-(-x // BLOCK) for x in ctx))
    c.tables = torch.randint(0, SHARED, (len(nodes), width), generator=g).int()
    blocks = SHARED
    owned = {}
    for s, (m, n) in enumerate(zip(nodes, ctx)):
        for b in range(max(n - m, 0) // BLOCK, -(-n // BLOCK)):
            c.tables[s, b] = blocks
            owned[blocks] = min(BLOCK, n - b * BLOCK)
            blocks += 1
    shape = (blocks, 2, BLOCK, hkv, dim)
    c.k_scale = c.v_scale = None
    if kv == "same":
        k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    else:
        k, v = ((torch.randn(shape, generator=g) * 60).clamp(-448, 448).to(FP8) for _ in range(2))
        if kv == "fp8":
            c.k_scale, c.v_scale = torch.tensor(1 / 60.0), torch.tensor(1 / 50.0)
        else:
            c.k_scale, c.v_scale = ((torch.rand(shape[:-1], generator=g) + 0.5)[:, 1] / 60 for _ in range(2))
    c.k, c.v = k[:, 1], v[:, 1]
    for b, n in owned.items():
        for x in (c.k, c.v) + ((c.k_scale, c.v_scale) if kv == "fp8_vector" else ()):
            x[b, n:] = torch.full_like(x[b, n:], math.nan, dtype=torch.float32).to(x.dtype)
    c.q = (torch.randn(sum(nodes), hq, dim, generator=g) * 1.5).to(dtype)
    c.lengths = torch.tensor(ctx, dtype=torch.int32)
    c.cu = torch.tensor(np.concatenate([[0], np.cumsum(nodes)]), dtype=torch.int32)
    c.max_q = max(nodes)
    c.bits = [ancestor_bits(random_parents(m - 1, g)) if m else [] for m in nodes]
    c.mask = pack_bits([b for rows in c.bits for b in rows], -(-c.max_q // 64))
    return c


def kv_waves(c):
    """kv groups of a workgroup: four waves over the row waves that hold a kv head's rows."""
    rows = c.max_q * (c.q.shape[1] // c.k.shape[2])
    return 4 if rows <= 32 else 2 if rows <= 64 else 1


def tiles_apart(c, window):
    """32-position tiles of all (sequence, group of neighbouring heads, row block) of the call."""
    group, hkv, kw = c.q.shape[1] // c.k.shape[2], c.k.shape[2], kv_waves(c)
    total = 0
    for m, n in zip(c.nodes, c.ctx):
        first = max(0, n - m - window) if window else 0
        total += (-(-n // 32) - first // 32) * -(-m * group // (32 * (4 // kw))) * -(-hkv // kw)
    return total


def lengths_of(count, tree, longest, seed):
    """Trees of 1 .. ``tree`` nodes over contexts from the tree alone to ``longest``; a sequence
    without rows and one without keys."""
    r = np.random.default_rng(seed)
    nodes = [int(x) for x in r.integers(1, tree + 1, count)]
    nodes[1], nodes[2], nodes[3] = tree, 0, tree
    ctx = [m + int(x) for m, x in zip(nodes, r.integers(longest // 4, longest, count))]
    ctx[3], ctx[4] = tree, nodes[4]
    ctx[-1] = longest + tree
    return nodes, ctx


# (sequences, most nodes, longest prefix, q heads, kv heads, dim, type, kv, window)
BATCHES = [
    # four kv groups
    (70, 16, 2200, 10, 5, 128, BF, "same", 0),         # 4 + 1 heads
    (70, 16, 2200, 16, 8, 128, BF, "fp8", 0),
    (70, 30, 2200, 7, 7, 64, HF, "fp8_vector", 0),      # 4 + 3
    (70, 16, 2200, 12, 6, 96, BF, "same", 0),
    (70, 16, 2200, 12, 6, 96, HF, "fp8_vector", 0),
    (70, 16, 2200, 6, 6, 64, HF, "same", 0),
    (70, 16, 2200, 4, 2, 256, BF, "fp8", 0),            # 2 heads of four groups
    (50, 7, 2200, 20, 5, 256, HF, "fp8_vector", 0),
    (130, 16, 3000, 16, 8, 128, BF, "fp8_vector", 700),
    # two
    (60, 16, 2200, 20, 5, 128, BF, "same", 0),
    (60, 32, 2600, 10, 5, 128, HF, "fp8_vector", 0),
    (40, 64, 2200, 7, 7, 96, BF, "same", 0),
    (70, 40, 3000, 3, 3, 64, BF, "fp8_vector", 0),
    (60, 25, 2200, 6, 3, 256, BF, "fp8", 0),
    (60, 40, 2600, 5, 5, 64, HF, "same", 900),
]


def batch(count, tree, longest, hq, hkv, dim, dtype, kv, window):
    nodes, ctx = lengths_of(count, tree, longest, seed=dim + hkv)
    c = make_batch(nodes, ctx, hq, hkv, dim, dtype, kv, seed=count + dim)
    # the count from which the groups go apart: 8 tiles for each of the launch's workgroups
    assert hkv > 1 and kv_waves(c) > 1 and tiles_apart(c, window) >= 8 * (256 if dim == 256 else 512)
    return c


@pytest.mark.parametrize("count,tree,longest,hq,hkv,dim,dtype,kv,window", BATCHES)
def test_heads_apart(pkg, dev, count, tree, longest, hq, hkv, dim, dtype, kv, window):
    c = batch(count, tree, longest, hq, hkv, dim, dtype, kv, window)
    got = attend(pkg, dev, c, window=window)
    want, tol = dense(c, window)
    over = (got.double().cpu() - want).abs() - tol
    assert torch.isfinite(got).all() and over.max() <= 0, float(over.max())
    assert torch.equal(attend(pkg, dev, c, window=window), got)
    if kv != "fp8":
        comp = attend(pkg, dev, c, pkg.MI355XPagedAttention(compensate=True), window=window)
        want, tol = dense(c, window, second=True)
        over = (comp.double().cpu() - want).abs() - tol
        assert torch.isfinite(comp).all() and over.max() <= 0, float(over.max())


@pytest.mark.parametrize("count,tree,longest,hq,hkv,dim,dtype,kv,window",
                         [BATCHES[i] for i in (0, 2, 5, 7, 8, 9, 10, 11, 14)])
def test_hidden_values_apart(pkg, dev, count, tree, longest, hq, hkv, dim, dtype, kv, window):
    """NaN and infinities of the last kv head at tree positions that some rows do not see: a value
    shows in the rows that see it, in its dim only; a key of the first head in their whole rows."""
    c = batch(count, tree, longest, hq, hkv, dim, dtype, kv, window)
    clean, tol = dense(c, window)
    group, at = hq // hkv, dim - 3
    hit = torch.zeros(c.q.shape[0], dtype=torch.bool)
    for s, (m, n) in enumerate(zip(c.nodes, c.ctx)):
        if m < 3 or s % 3 == 0:
            continue
        vis = sees(c, s, window)
        for i, node in enumerate((m // 2, m - 1)):
            pos = n - m + node
            blk, off = int(c.tables[s, pos // BLOCK]), pos % BLOCK
            assert blk >= SHARED
            bad = torch.tensor(math.nan if kv != "same" or i else -math.inf)
            c.v[blk, off, hkv - 1, at] = bad.to(c.v.dtype)
            c.k[blk, off, 0, at] = torch.tensor(math.nan).to(c.k.dtype)
            hit[int(c.cu[s]):int(c.cu[s + 1])] |= vis[:, pos]
    assert hit.any() and not hit.all()
    got = attend(pkg, dev, c, window=window).double().cpu()
    over = (got[~hit] - clean[~hit]).abs() - tol[~hit]
    assert torch.isfinite(got[~hit]).all() and over.max() <= 0
    last = slice(hq - group, hq)
    assert not torch.isfinite(got[hit][:, last, at]).any()
    rest = [d for d in range(dim) if d != at]
    for heads in (slice(group, hq - group), last):
        dims = rest if heads is last else list(range(dim))
        a, b, t = (x[hit][:, heads][..., dims] for x in (got, clean, tol))
        assert torch.isfinite(a).all() and ((a - b).abs() <= t).all()
    assert torch.isnan(got[hit][:, :group]).all()
