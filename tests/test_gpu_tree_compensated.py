"""Tree attention with the compensated product of weights and values."""

import math

import pytest
import torch

from tests.test_gpu_tree_edges import attend, close
from tests.tree_cases import make_case
from tests.tree_dense import dense

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


# (nodes, ctx, q heads, kv heads, dim, type, kv, block size, window)
@pytest.mark.parametrize("nodes,ctx,hq,hkv,dim,dtype,kv,block,window", [
    ([1, 5], [700, 33], 4, 4, 128, BF, "same", 16, 0),
    ([16, 3, 32], [515, 64, 32], 2, 2, 64, BF, "same", 16, 0),
    ([16, 16], [300, 1025], 8, 2, 128, BF, "same", 16, 0),
    ([26, 9], [260, 511], 16, 4, 128, BF, "same", 32, 0),
    ([12, 40], [100, 333], 5, 5, 96, BF, "same", 16, 0),
    ([9, 20], [257, 96], 2, 2, 256, BF, "same", 16, 0),
    ([33, 70], [129, 400], 8, 2, 128, HF, "same", 16, 0),
    ([16, 7], [515, 96], 16, 8, 128, BF, "fp8", 16, 0),
    ([30, 50], [515, 96], 8, 4, 128, BF, "fp8_vector", 16, 0),
    ([12, 31], [300, 77], 4, 2, 64, HF, "fp8_vector", 16, 0),
    ([50, 31], [300, 77], 4, 2, 64, HF, "fp8", 16, 0),
    ([44], [300], 10, 2, 96, BF, "fp8", 16, 0),
    ([30], [300], 4, 1, 256, BF, "fp8_vector", 16, 0),
    ([16, 20], [515, 96], 4, 2, 128, BF, "same", 16, 100),
    ([256], [2300], 2, 1, 64, BF, "same", 8, 0),
    ([200, 1], [3200, 1], 4, 1, 128, BF, "same", 24, 0),
    ([16, 7], [200, 96], 4, 2, 128, BF, "same", 12, 0),   # the vector form: float32 weights
    ([9, 20], [50, 80], 2, 1, 80, HF, "fp8", 5, 0),
    ([16, 7], [215, 96], 4, 2, 64, F32, "same", 16, 0),
])
def test_weights_of_twice_the_bits(pkg, dev, nodes, ctx, hq, hkv, dim, dtype, kv, block, window):
    c = make_case(nodes, ctx, hq, hkv, dim, dtype, kv, block, seed=sum(nodes) + dim)
    got = attend(pkg, dev, c, pkg.MI355XPagedAttention(compensate=True), window=window)
    close(got, *dense(c, window, second=dtype != F32))


@pytest.mark.parametrize("d,nodes", [(256, 1), (128, 1), (128, 40), (64, 70)])
def test_small_value_residual(pkg, dev, d, nodes):
    """Two positions whose weighted values nearly cancel, which weights of 8 bits lose: within
    5e-6 of the float64 closed form, as the packed causal form gives them."""
    s1 = {256: 16.0, 128: 11.3125, 64: 8.0}[d] * -0.5 / math.sqrt(d)
    c = make_case([nodes], [nodes + 2], 1, 1, d, BF, seed=1, bits=[[0] * nodes])
    c.q.fill_(0)
    c.q[..., 0] = {256: 16.0, 128: 11.3125, 64: 8.0}[d]
    c.k.fill_(0)
    c.v.fill_(0)
    blk = int(c.tables[0, 0])
    c.k[blk, 1, 0, 0] = -0.5
    c.v[blk, 0, 0, 0], c.v[blk, 1, 0, 0] = -0.60546875, 1
    w0, w1 = 1 / (1 + math.exp(s1)), math.exp(s1) / (1 + math.exp(s1))
    expected = w0 * -0.60546875 + w1
    assert abs(expected) > 0.0003
    got = attend(pkg, dev, c, pkg.MI355XPagedAttention(compensate=True))
    assert ((got[..., 0].double() - expected).abs() <= 5e-6).all() and (got[..., 1:] == 0).all()
    plain = attend(pkg, dev, c)
    assert ((plain[..., 0].double() - expected).abs() > 5e-6).all()


def test_the_backends_choice_reaches_trees(pkg, dev):
    """``create_backend(packed_window_shape=...)`` says that weights are compensated: a chain of
    nodes is as near to float64 as the causal window, in a graph too, and twice the same."""
    nodes, ctx = [5, 5, 3], [300, 1030, 77]
    c = make_case(nodes, ctx, 16, 4, 128, BF, seed=20, bits=[[(2 << i) - 1 for i in range(m)] for m in nodes])
    backend = pkg.create_backend("auto", dev, BF, 128, 16, packed_window_shape=object())
    assert backend.info["compensated_p"]
    want, tol = dense(c, second=True)
    args = [x.to(dev) for x in (c.q, c.k, c.v, c.tables, c.lengths, c.cu)]
    mask = c.mask.to(dev)
    first = backend.tree(*args, c.max_q, mask)
    close(first, want, tol)
    close(backend.prefill(*args, c.max_q), want, tol)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = backend.tree(*args, c.max_q, mask)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
        assert math.isfinite(torch.randn(1 << 16, device=dev).sum().item())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinite_value_scales_stay_infinite(pkg, dev, dtype):
    """An infinite scale of a visible value, whose product with a weight has no dropped part: the
    rows that see it hold infinities, the others numbers, as without compensation."""
    c = make_case([16, 9], [200, 131], 4, 2, 64, dtype, "fp8_vector", seed=3)
    blk = int(c.tables[0, 3])
    c.v_scale[blk, 5, 0] = math.inf  # position 53 of sequence 0, kv head 0
    c.v[blk, 5, 0] = torch.full((64,), 2.0).to(c.v.dtype)
    got = attend(pkg, dev, c, pkg.MI355XPagedAttention(compensate=True)).float().cpu()
    assert torch.isposinf(got[:16, :2]).all()
    assert torch.isfinite(got[:16, 2:]).all() and torch.isfinite(got[16:]).all()
    assert torch.equal(torch.isposinf(attend(pkg, dev, c).float().cpu()), torch.isposinf(got))


@pytest.mark.parametrize("hq,hkv,dim,nodes", [(2, 2, 128, [16, 7]), (4, 1, 64, [40, 12]), (8, 2, 96, [9, 16])])
@pytest.mark.parametrize("low,high", [(-26, -22), (-20, 4), (2, 6)])
def test_value_scales_of_any_size(pkg, dev, hq, hkv, dim, nodes, low, high):
    """fp16 rows over per-vector scales far from 1, and over scales that differ widely: what the
    rounding of weight times scale drops is held over the same power of two."""
    c = make_case(nodes, [515, 96], hq, hkv, dim, HF, "fp8_vector", seed=50 + dim)
    g = torch.Generator().manual_seed(dim)
    exps = low + (high - low) * torch.rand(c.v_scale.shape, generator=g)
    c.v_scale = torch.where(c.v_scale.isnan(), c.v_scale, torch.exp2(exps))
    close(attend(pkg, dev, c, pkg.MI355XPagedAttention(compensate=True)), *dense(c, second=True))


@pytest.mark.parametrize("dtype,kv,dim", [(BF, "same", 128), (BF, "fp8_vector", 64), (HF, "same", 96)])
def test_hidden_values_with_compensation(pkg, dev, dtype, kv, dim):
    """NaN at the last node's position: only that node's row of its kv head shows it, in its dim."""
    nodes, ctx = [16, 40], [200, 131]
    c = make_case(nodes, ctx, 4, 2, dim, dtype, kv, seed=3)
    want, tol = dense(c, second=True)
    rows = []
    for s in range(2):
        blk, off = int(c.tables[s, (ctx[s] - 1) // c.block]), (ctx[s] - 1) % c.block
        c.v[blk, off, 0, dim // 2] = torch.tensor(math.nan).to(c.v.dtype)
        rows.append(int(c.cu[s + 1]) - 1)
    got = attend(pkg, dev, c, pkg.MI355XPagedAttention(compensate=True)).double().cpu()
    hit = torch.zeros_like(want, dtype=torch.bool)
    for r in rows:
        hit[r, :2, dim // 2] = True
    assert torch.isnan(got[hit]).all() and torch.isfinite(got[~hit]).all()
    assert ((got - want).abs() <= tol)[~hit].all()
