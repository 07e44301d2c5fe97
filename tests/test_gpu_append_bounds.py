"""Appends, loads and rotations at the bounds of their arguments: windows longer than ``max_seqlen_q``, and
calls whose padded windows or rows are more than one launch holds (2^32 threads)."""

import pytest
import torch

from oracle import rotary as orot
from tests.test_gpu_append import POOLS, Round, _equal, _layer, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", POOLS)
def test_windows_longer_than_their_bound(pkg, dev, kind):
    """The first ``max_seqlen_q`` rows of a longer window go to, turn by and come back from the places that
    they have in the whole window; the rows behind them are left."""
    _say("longer", kind)
    plan = pkg.Rotary(64, device=dev)
    r = Round(kind, torch.bfloat16, 16, 2, 64, [30, 0, 7, 13], [20, 40, 5, 3], seed=41, hq=4)
    bound, counts = 7, r.counts
    r.counts = [min(n, bound) for n in counts]  # (run takes the largest)
    begins = r.cu[:-1].tolist()
    kept = torch.cat([torch.arange(b, b + n) for b, n in zip(begins, r.counts)])
    got = r.run(pkg, dev)
    want = []
    for pool, scale, rows in ((r.k, r.ks, r.new_k), (r.v, r.vs, r.new_v)):
        pool, scale = pool.clone(), None if scale is None else scale.clone()
        ends = [n - c + m for n, c, m in zip(r.lengths, counts, r.counts)]
        orot.append(_layer(pool), _layer(scale), rows[kept].float(), r.tables, ends, r.counts)
        want.append((pool, scale))
    _equal(got, want)
    turned = r.run(pkg, dev, plan)[4]
    alone, _ = pkg.apply_rotary(r.q.to(dev), None, r.places.to(dev), plan)
    assert torch.equal(turned[kept], alone.cpu()[kept])
    # read back with the same bound
    k, v, ks, vs = (None if x is None else _layer(x).to(dev) for x in got[:4])
    lengths = torch.tensor(r.lengths, dtype=torch.int32, device=dev)
    a, b = pkg.load_kv(k, v, r.tables.to(dev), lengths, r.cu.to(dev), bound, len(r.places), ks, vs,
                       dtype=torch.float32)
    for x, (pool, scale) in zip((a, b), want):
        whole = orot.load(_layer(pool), _layer(scale), r.tables, r.lengths, counts)
        assert torch.equal(x.cpu()[kept], whole.float()[kept])


@pytest.mark.parametrize("kind", ("same", "int8"))
def test_padded_windows_past_one_launch(pkg, dev, kind):
    """One long window beside a thousand single tokens: 2^24 tiles of 256 threads, nearly all without rows."""
    _say("past one launch", kind)
    # (tiles of 8 rows; blocks of 8 tokens)
    n, long = 1040, (1 << 17) + 8
    bs, rows = 8, n - 1 + long
    g = torch.Generator(device=dev).manual_seed(42)
    counts = torch.ones(n, dtype=torch.int32, device=dev)
    counts[n - 2] = long  # (a place past the first launch's)
    cu = torch.cat([counts.new_zeros(1), counts.cumsum(0).int()])
    width = long // bs
    blocks = width + n
    tables = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    tables[:, 0] = torch.arange(n, device=dev, dtype=torch.int32) + width
    tables[n - 2] = torch.arange(width, device=dev, dtype=torch.int32)
    dtype = torch.bfloat16 if kind == "same" else torch.int8
    k, v = (torch.zeros(blocks, bs, 1, 16, dtype=dtype, device=dev) for _ in range(2))
    ks, vs = (None, None) if kind == "same" else (torch.zeros(blocks, 1, device=dev) for _ in range(2))
    new_k, new_v = (torch.randn(rows, 1, 16, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    pkg.append_kv(k, v, new_k, new_v, tables, counts, cu, long, ks, vs)
    a, b = pkg.load_kv(k, v, tables, counts, cu, long, rows, ks, vs, dtype=torch.float32)
    for x, rows_in, scale in ((a, new_k, ks), (b, new_v, vs)):
        if kind == "same":
            assert torch.equal(x, rows_in.float())
        else:
            # half a step of the row's block, at most 127 of them, and two roundings of float32
            at = torch.cat([torch.full((1,), width + s, device=dev) if s != n - 2 else
                            torch.arange(long, device=dev) // bs for s in range(n)])
            near = scale[at][:, None] * (0.5 + 2.0 ** -15)
            assert ((x - rows_in.float()).abs() <= near).all()


def test_rotations_past_one_launch(pkg, dev):
    """2^27 rows and some: those at both ends and across the launches' borders as a call of them alone."""
    _say("rotations past one launch")
    plan = pkg.Rotary(2, device=dev)
    rows = (1 << 27) + 77
    q = torch.empty(rows, 1, 2, dtype=torch.bfloat16, device=dev).uniform_(-1, 1)
    pos = torch.arange(rows, device=dev)
    got = pkg.apply_rotary(q, None, pos, plan)[0]
    for at in (0, (1 << 26) - 100, (1 << 27) - 100, rows - 200):
        part = slice(at, at + 200)
        assert torch.equal(got[part], pkg.apply_rotary(q[part], None, pos[part], plan)[0])


@pytest.mark.parametrize("kind", ("fp8", "int8"))
@pytest.mark.parametrize("exponent", (-126, -120, -112, -100, -91, -90, -80, 0, 100))
def test_codes_of_values_at_the_middle_of_two(pkg, dev, kind, exponent):
    """Rows at and next to the border of two codes, over scales of any size: the division's codes, bit for bit,
    those of earlier rows among them where a block's scale grows."""
    _say("middle", kind, exponent)
    g = torch.Generator().manual_seed(200 + exponent)
    top = 127 if kind == "int8" else 448
    r = Round(kind, torch.float32, 16, 4, 64, [0, 5, 16, 3], [6, 9, 40, 1], seed=43)
    for name in ("new_k", "new_v"):
        # (scales of every mantissa: a row's largest value gives its block's, the same for all of its rows)
        most = (1 + torch.rand(1, 4, 1, generator=g)) * 2.0 ** exponent * top
        scale = most * torch.tensor(1.0 / top, dtype=torch.float32)
        shape = (len(r.places), 4, 64)
        if kind == "int8":
            middle = torch.randint(-126, 126, shape, generator=g) + 0.5
        else:
            step = 2.0 ** torch.randint(-9, 5, shape, generator=g)
            middle = (torch.randint(8, 15, shape, generator=g) + 0.5) * step
        x = (middle.double() * scale.double()).float()
        near = torch.randint(-1, 2, shape, generator=g, dtype=torch.int32)
        x = (x.view(torch.int32) + near).view(torch.float32)
        x[..., 0] = most[..., 0]
        setattr(r, name, x)
    for name in ("ks", "vs"):  # earlier tokens over a scale that grows, or does not
        held = getattr(r, name)
        held.fill_(2.0 ** max(exponent - 1, -126))
        held *= (1 + torch.rand(held.shape, generator=g)) * (0.7 if exponent > -126 else 1)
    _equal(r.run(pkg, dev), r.expect())
