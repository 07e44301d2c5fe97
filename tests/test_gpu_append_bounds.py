"""Appends and loads at the bounds of their arguments: windows longer than ``max_seqlen_q``."""

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
