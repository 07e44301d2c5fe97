"""Appends into the paged cache and its reading back, against ``oracle/rotary.py``."""

import math

import pytest
import torch

from oracle import rotary as orot

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
POOLS = ("same", "tensor", "vector", "fp8", "int8")


def _say(*args):
    print("[case]", *args, flush=True)


def _pool(kind, blocks, bs, heads, dim, dtype, g):
    """Two layers of which the second is used, and its scales."""
    shape = (blocks, 2, bs, heads, dim)
    if kind == "same":
        return torch.randn(shape, generator=g).to(dtype), None
    codes = (torch.randint(-127, 128, shape, generator=g).to(torch.int8) if kind == "int8" else
             (torch.randn(shape, generator=g) * 90).clamp(-448, 448).to(FP8))
    if kind == "tensor":
        return codes, torch.tensor(0.011)
    held = shape[:4] if kind == "vector" else (blocks, 2, heads)
    return codes, (torch.rand(held, generator=g) + 0.5) * 3 / (127 if kind == "int8" else 448)


def _layer(x):
    return None if x is None else x if x.ndim == 0 else x[:, 1]


def _bits(x):
    return x.contiguous().view(torch.uint8) if x.dtype in (FP8, torch.int8) else x


class Round:
    """One append: windows of counts[s] rows behind befores[s] cached positions."""

    def __init__(self, kind, dtype, bs, heads, dim, befores, counts, seed, hq=0, spare=1):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.counts = kind, counts
        self.lengths = [b + c for b, c in zip(befores, counts)]
        width = max(1, max(-(-n // bs) for n in self.lengths)) + spare
        blocks = len(counts) * width + 1
        self.tables = torch.randperm(blocks, generator=g)[:len(counts) * width].int().view(-1, width)
        self.k, self.ks = _pool(kind, blocks, bs, heads, dim, dtype, g)
        self.v, self.vs = _pool(kind, blocks, bs, heads, dim, dtype, g)
        rows = sum(counts)
        # row sizes differ, so that some raise their block's scale and some do not
        size = torch.rand(rows, heads, 1, generator=g) * 3 + 0.1
        self.new_k, self.new_v = ((torch.randn(rows, heads, dim, generator=g) * size).to(dtype)
                                  for _ in range(2))
        self.q = torch.randn(rows, hq, dim, generator=g).to(dtype) if hq else None
        self.cu = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
        self.places = torch.cat([torch.arange(n - c, n) for n, c in zip(self.lengths, counts)]).long()

    def run(self, pkg, dev, rotary=None, positions=None, **kw):
        """(k, v, ks, vs, q') on the host, of copies on the device."""
        k, v = self.k.to(dev), self.v.to(dev)
        ks, vs = (None if x is None else x.to(dev) for x in (self.ks, self.vs))
        q = pkg.append_kv(_layer(k), _layer(v), self.new_k.to(dev), self.new_v.to(dev),
                          self.tables.to(dev), torch.tensor(self.lengths, dtype=torch.int32, device=dev),
                          self.cu.to(dev), max(self.counts), _layer(ks), _layer(vs), rotary=rotary,
                          positions=positions, q=None if self.q is None else self.q.to(dev), **kw)
        return [None if x is None else x.cpu() for x in (k, v, ks, vs, q)]

    def expect(self):
        out = []
        for pool, scale, rows in ((self.k, self.ks, self.new_k), (self.v, self.vs, self.new_v)):
            pool, scale = pool.clone(), None if scale is None else scale.clone()
            orot.append(_layer(pool), _layer(scale), rows.float(), self.tables, self.lengths, self.counts)
            out.append((pool, scale))
        return out


def _equal(got, want):
    for (pool, scale), g, s in zip(want, got[:2], got[2:4]):
        assert torch.equal(_bits(g), _bits(pool))
        assert (s is None and scale is None) or torch.equal(s, scale)


RAGGED = ([0, 3, 16, 37, 100], [1, 20, 5, 64, 3])


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("bs,heads,dim", [(16, 4, 128), (16, 1, 64), (8, 3, 96), (64, 2, 256), (3, 2, 7),
                                          (40, 2, 80)])
def test_unrotated_appends_are_exact(pkg, dev, kind, dtype, bs, heads, dim):
    """Codes, scales and every byte of the pool that is not written, bit for bit."""
    _say("append", kind, dtype, bs, heads, dim)
    r = Round(kind, dtype, bs, heads, dim, *RAGGED, seed=bs + dim)
    _equal(r.run(pkg, dev), r.expect())


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("dim,rot,interleaved", [(128, 128, False), (128, 64, True), (96, 96, False),
                                                 (64, 48, True), (80, 20, False), (256, 128, False)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_rotated_appends(pkg, dev, kind, dim, rot, interleaved, dtype):
    """Every cached number against the rotation in float64: the rotation's float32 error, half a
    step of the pool's type or codes, and for codes that were held over a larger scale half
    a step of theirs; q as ``apply_rotary`` gives it, bit for bit."""
    _say("rotated", kind, dim, rot, interleaved, dtype)
    plan = pkg.Rotary(rot, interleaved=interleaved, device=dev)
    r = Round(kind, dtype, 16, 2, dim, *RAGGED, seed=dim, hq=6)
    k, v, ks, vs, q = r.run(pkg, dev, plan)
    alone, _ = pkg.apply_rotary(r.q.to(dev), None, r.places.to(dev), plan)
    assert torch.equal(q, alone.cpu())
    turns = plan.turns.cpu()
    rows = orot.rotate(r.new_k, r.places, turns, 1.0, interleaved)
    near = orot.rotate_error(r.new_k, turns, 1.0, interleaved)
    # values do not turn: exact, as without a rotation
    want_v = r.expect()[1]
    assert torch.equal(_bits(v), _bits(want_v[0])) and (vs is None or torch.equal(vs, want_v[1]))
    pool, scale = _layer(k), _layer(ks)
    got = orot.load(pool, scale, r.tables, r.lengths, r.counts)
    if kind == "same":
        step = (rows.abs() + near) * torch.finfo(dtype).eps / 2
    else:
        f = torch.stack([
            torch.full((2,), float(scale), dtype=torch.float64) if scale.ndim == 0 else
            (scale[int(r.tables[s, p // 16]), p % 16] if scale.ndim == 3 else
             scale[int(r.tables[s, p // 16])]).double()
            for s, (n, c) in enumerate(zip(r.lengths, r.counts)) for p in range(n - c, n)])[..., None]
        # a code is off by half a step: 0.5 of int8's, 2^-4 of an e4m3 value or 2^-10; the division
        # by the scale by 2^-24, and a scale of the call by the rotation's and its own rounding
        step = f * 0.5 if kind == "int8" else torch.maximum(rows.abs() * 2.0 ** -4, f * 2.0 ** -10)
        step = step * (1 + 2.0 ** -16) + rows.abs() * 2.0 ** -20
        if kind == "tensor":
            clipped = rows.clamp(-448 * f, 448 * f)
            near, rows = near + 0, clipped
    assert ((got - rows).abs() <= near + step).all()
    if kind in ("fp8", "int8"):
        # earlier tokens of a block that was gone on with
        before = [n - c for n, c in zip(r.lengths, r.counts)]
        tails = [b % 16 for b in before]
        old = orot.load(_layer(r.k), _layer(r.ks), r.tables, before, tails)
        new = orot.load(pool, scale, r.tables, before, tails)
        f = torch.cat([scale[int(r.tables[s, b // 16])].double().expand(t, -1)
                       for s, (b, t) in enumerate(zip(before, tails)) if t])[..., None]
        step = f * 0.5 if kind == "int8" else torch.maximum(old.abs() * 2.0 ** -4, f * 2.0 ** -10)
        assert ((new - old).abs() <= step * (1 + 2.0 ** -16)).all()


def test_many_heads_and_long_blocks(pkg, dev):
    """More heads than a workgroup's waves, blocks of more rows than a wave holds."""
    _say("many heads")
    for kind in ("fp8", "int8"):
        _equal(*(lambda r: (r.run(pkg, dev), r.expect()))(
            Round(kind, torch.bfloat16, 128, 55, 96, [5, 200], [200, 130], seed=9)))


def test_a_batch_of_windows_fills_the_grid(pkg, dev):
    _say("batch")
    g = torch.Generator().manual_seed(5)
    counts = torch.randint(0, 40, (300,), generator=g).tolist()
    befores = torch.randint(0, 50, (300,), generator=g).tolist()
    r = Round("int8", torch.bfloat16, 16, 1, 64, befores, counts, seed=6)
    _equal(r.run(pkg, dev), r.expect())


def test_explicit_positions(pkg, dev):
    """Rows that turn by other positions than their places, as the nodes of a tree do."""
    _say("positions")
    plan = pkg.Rotary(64, device=dev)
    r = Round("same", torch.float32, 16, 2, 64, [10], [6], seed=7, hq=4)
    pos = torch.tensor([10, 11, 11, 12, 12, 13])
    k, _, _, _, q = r.run(pkg, dev, plan, positions=pos.to(dev))
    want = pkg.apply_rotary(r.q.to(dev), r.new_k.to(dev), pos.to(dev), plan)
    assert torch.equal(q, want[0].cpu())
    got = orot.load(k[:, 1], None, r.tables, [16], [6])
    assert torch.equal(got, want[1].cpu().double())


@pytest.mark.parametrize("kind", POOLS)
def test_rows_without_a_place_are_not_written(pkg, dev, kind):
    """Positions before 0 or past the table and entries outside the pool: nothing is written,
    q is turned; rows of no sequence and rows past max_seqlen_q are left."""
    _say("no place", kind)
    plan = pkg.Rotary(64, device=dev)
    r = Round(kind, torch.bfloat16, 16, 2, 64, [20, 0, 5, 3], [20, 9, 30, 4], seed=8, hq=2, spare=0)
    r.lengths[1] = 4            # five rows before position 0
    r.tables = r.tables.clone()
    r.tables[0, 2], r.tables[3, 0] = -1, r.k.shape[0] + 7
    r.tables = r.tables[:, :2].contiguous()  # sequence 2 ends at 35, the table at 32
    r.places = torch.cat([torch.arange(n - c, n) for n, c in zip(r.lengths, r.counts)])
    got = r.run(pkg, dev)
    _equal(got, r.expect())
    got = r.run(pkg, dev, plan)
    alone, _ = pkg.apply_rotary(r.q.to(dev), None, r.places.to(dev), plan)
    assert torch.equal(got[4], alone.cpu())
    # (reading places that hold nothing gives zeros)
    ks, vs = (None if x is None else _layer(x).to(dev) for x in got[2:4])
    lengths = torch.tensor(r.lengths, dtype=torch.int32, device=dev)
    a, b = pkg.load_kv(_layer(got[0].to(dev)), _layer(got[1].to(dev)), r.tables.to(dev), lengths,
                       r.cu.to(dev), 30, len(r.places), ks, vs, dtype=torch.float32)
    for x, pool, scale in ((a, got[0], got[2]), (b, got[1], got[3])):
        want = orot.load(_layer(pool), _layer(scale), r.tables, r.lengths, r.counts)
        assert torch.equal(x.cpu(), want.float())


def test_special_values(pkg, dev):
    """What is not finite does not move a block's scale: e4m3 keeps NaN and clamps infinities,
    int8 takes NaN as 0; a block of zeros has the smallest scale, one of NaN alone too."""
    _say("special")
    for kind in ("fp8", "int8"):
        r = Round(kind, torch.float32, 16, 2, 64, [0, 4], [3, 3], seed=11)
        r.new_k[0, 0, 5], r.new_k[1, 0, 6], r.new_k[4, 1, 7] = float("nan"), float("inf"), -float("inf")
        r.new_v[:3] = 0
        r.new_v[3:, 0] = float("nan")
        got = r.run(pkg, dev)
        want = r.expect()
        for g, (pool, scale) in zip(got[:2], want):
            a, b = _layer(g).float(), _layer(pool).float()
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
        assert torch.equal(got[2], want[0][1]) and torch.equal(got[3], want[1][1])
        assert got[3][int(r.tables[0, 0]), 1, 0] == 2.0 ** -126


def test_tiny_and_huge_values(pkg, dev):
    """Scales at both ends of float32."""
    _say("tiny")
    for kind in ("vector", "fp8", "int8"):
        r = Round(kind, torch.float32, 16, 2, 64, [0, 2], [5, 5], seed=12)
        r.new_k *= 1e-37
        r.new_v *= 1e37
        _equal(r.run(pkg, dev), r.expect())


@pytest.mark.parametrize("exponent", (-140, -126, -91, -90, -60, 60, 119, 120, 121, 126))
def test_given_scales_at_both_ends(pkg, dev, exponent):
    """Codes over one scale that is given are ``store_fp8``'s: values about, far above and far
    below it, zeros of both signs, infinities and NaN."""
    _say("given", exponent)
    for sign in (1.0, -1.0):
        r = Round("tensor", torch.float32, 16, 2, 64, [0, 2], [5, 5], seed=14)
        r.ks = r.vs = torch.tensor(sign * 1.37 * 2.0 ** exponent)
        for x in (r.new_k, r.new_v):
            x *= float(r.ks) * 90
            x[0, 0, :9] = torch.tensor([0.0, -0.0, 3e38, -3e38, 1e-44, -1e-44, math.inf, -math.inf, math.nan])
        got = r.run(pkg, dev)
        k, v = (_layer(x).to(dev) for x in (r.k, r.v))
        scales = torch.zeros(k.shape[:3], device=dev)
        blocks = r.tables[torch.repeat_interleave(torch.arange(2), torch.tensor(r.counts)), r.places // 16]
        pkg.store_fp8(r.new_k.to(dev), r.new_v.to(dev), k, v, scales, scales.clone(), blocks.long().to(dev),
                      (r.places % 16).to(dev), 448.0, fixed_scale=float(r.ks))
        for a, b in zip(got[:2], (k, v)):
            assert torch.equal(_bits(_layer(a)), _bits(b).cpu())


def test_repeated_single_tokens(pkg, dev):
    """A sequence grown token by token, over several blocks, in place on the device."""
    _say("token by token")
    for kind in ("fp8", "int8"):
        g = torch.Generator().manual_seed(13)
        pools = [_pool(kind, 4, 8, 2, 64, torch.bfloat16, g) for _ in range(2)]
        host = [(p.clone(), s.clone()) for p, s in pools]
        (k, ks), (v, vs) = [(p.to(dev), s.to(dev)) for p, s in pools]
        tables = torch.tensor([[2, 0, 3]], dtype=torch.int32)
        for n in range(1, 21):
            a, b = (torch.randn(1, 2, 64, generator=g).to(torch.bfloat16) * (1 + n % 5) for _ in range(2))
            pkg.append_kv(k[:, 1], v[:, 1], a.to(dev), b.to(dev), tables.to(dev),
                          torch.tensor([n], dtype=torch.int32, device=dev),
                          torch.tensor([0, 1], dtype=torch.int32, device=dev), 1, ks[:, 1], vs[:, 1])
            for (p, s), x in zip(host, (a, b)):
                orot.append(p[:, 1], s[:, 1], x.float(), tables, [n], [1])
        assert torch.equal(_bits(k.cpu()), _bits(host[0][0])) and torch.equal(ks.cpu(), host[0][1])
        assert torch.equal(_bits(v.cpu()), _bits(host[1][0])) and torch.equal(vs.cpu(), host[1][1])


def test_unaligned_pools_and_rows(pkg, dev):
    """Odd strides and offsets of rows, pools and scales take the elementwise form: the same bits."""
    _say("unaligned")
    for kind in ("same", "fp8", "int8", "vector"):
        r = Round(kind, torch.bfloat16, 16, 2, 64, [3, 18], [9, 17], seed=14)
        want = r.expect()
        blocks = r.k.shape[0]

        def loose(x):  # [blocks, 16, 2, 64] with rows of 65
            out = torch.zeros(blocks * 16 * 2 * 65 + 1, dtype=x.dtype, device=dev)[1:]
            out = out.view(blocks, 16, 2, 65)[..., :64]
            out.view(torch.uint8 if x.element_size() == 1 else torch.int16).copy_(
                x.to(dev).view(torch.uint8 if x.element_size() == 1 else torch.int16))
            return out

        k, v = loose(r.k[:, 1].contiguous()), loose(r.v[:, 1].contiguous())
        ks, vs = (None if x is None else _layer(x).to(dev).contiguous() for x in (r.ks, r.vs))
        pad = torch.zeros(26, 2, 67, dtype=torch.bfloat16, device=dev)
        nk, nv = pad[..., 3:], pad.clone()[..., 1:65]
        nk.copy_(r.new_k)
        nv.copy_(r.new_v)
        pkg.append_kv(k, v, nk, nv, r.tables.to(dev),
                      torch.tensor(r.lengths, dtype=torch.int32, device=dev), r.cu.to(dev), 17, ks, vs)
        assert torch.equal(_bits(k.cpu()), _bits(want[0][0][:, 1]))
        assert torch.equal(_bits(v.cpu()), _bits(want[1][0][:, 1]))
        if ks is not None:
            assert torch.equal(ks.cpu(), want[0][1][:, 1]) and torch.equal(vs.cpu(), want[1][1][:, 1])


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("dim,bs", [(128, 16), (96, 8), (7, 3), (64, 64)])
def test_load(pkg, dev, kind, dim, bs):
    """Element or code times scale in float32, rounded once to the asked type: the same bits."""
    _say("load", kind, dim, bs)
    r = Round(kind, torch.bfloat16, bs, 3, dim, [0, 5, 90, 33], [0, 1, 70, 33], seed=15)
    for dtype in (torch.float32, torch.float16, torch.bfloat16, None):
        got = pkg.load_kv(_layer(r.k).to(dev), _layer(r.v).to(dev), r.tables.to(dev),
                          torch.tensor(r.lengths, dtype=torch.int32, device=dev), r.cu.to(dev), 70,
                          104, *(None if x is None else _layer(x).to(dev) for x in (r.ks, r.vs)), dtype=dtype)
        for x, pool, scale in zip(got, (r.k, r.v), (r.ks, r.vs)):
            want = orot.load(_layer(pool), _layer(scale), r.tables, r.lengths, r.counts)
            assert x.dtype == (dtype or torch.bfloat16)
            # (an element of a row's type is exact; a product is rounded to float32, then to the type)
            assert torch.equal(x.cpu(), want.float().to(x.dtype))


def test_captured_appends_replay(pkg, dev):
    """A captured append reads lengths, tables, rows and pools anew at every replay."""
    _say("graph")
    plan = pkg.Rotary(64, device=dev)
    g = torch.Generator().manual_seed(16)
    pools = [_pool("int8", 9, 16, 2, 64, torch.bfloat16, g) for _ in range(2)]
    (k, ks), (v, vs) = [(p.to(dev), s.to(dev)) for p, s in pools]
    eager = [x.clone() for x in (k, v, ks, vs)]
    tables = torch.randperm(8, generator=g).int().view(2, 4).to(dev)
    lengths = torch.zeros(2, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device=dev)
    rows = [torch.zeros(3, h, 64, dtype=torch.bfloat16, device=dev) for h in (2, 2, 4)]

    def call(a, b, c, d):
        return pkg.append_kv(a[:, 1], b[:, 1], rows[0], rows[1], tables, lengths, cu, 2, c[:, 1], d[:, 1],
                             rotary=plan, q=rows[2])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(*(x.clone() for x in eager))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(k, v, ks, vs)
    for step in range(6):
        lengths.copy_(torch.tensor([2 * step + 2, step + 1]))
        for x in rows:
            x.copy_(torch.randn(x.shape, generator=g) * (1 + step))
        graph.replay()
        want = call(*eager)
        assert torch.equal(q, want)
        for a, b in zip((k, v, ks, vs), eager):
            assert torch.equal(_bits(a), _bits(b))


@pytest.mark.parametrize("kind", POOLS)
def test_a_longest_window_known_by_its_bound_only(pkg, dev, kind):
    """``max_seqlen_q`` far above the rows: the same pools, and the same numbers read back."""
    _say("bound", kind)
    r = Round(kind, torch.bfloat16, 16, 2, 64, [0, 37, 5], [3, 40, 0], 31)
    want, most = r.run(pkg, dev), max(r.counts)
    for bound in (4096, 2 ** 31 - 1):
        r.counts = [*r.counts[:2], bound]  # (run takes the largest)
        got = r.run(pkg, dev)
        r.counts[2] = 0
        for a, b in zip(want, got):
            assert (a is None) == (b is None) and (a is None or torch.equal(_bits(a), _bits(b)))
        k, v, ks, vs = (None if x is None else x.to(dev) for x in got[:4])
        rest = (r.tables.to(dev), torch.tensor(r.lengths, dtype=torch.int32, device=dev), r.cu.to(dev))
        loads = [pkg.load_kv(_layer(k), _layer(v), *rest, n, 43, _layer(ks), _layer(vs)) for n in (most, bound)]
        assert all(torch.equal(a, b) for a, b in zip(*loads))


def test_another_stream(pkg, dev):
    _say("stream")
    r = Round("int8", torch.bfloat16, 16, 4, 128, *RAGGED, seed=17)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = r.run(pkg, dev)
    _equal(got, r.expect())


def test_refusals(pkg, dev):
    i32 = dict(dtype=torch.int32, device=dev)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev)
    k, v = (torch.zeros(4, 16, 2, 64, dtype=torch.int8, device=dev) for _ in range(2))
    s, t = (torch.ones(4, 2, device=dev) for _ in range(2))
    tables, lengths, cu = torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32)
    ok = dict(key_cache=k, value_cache=v, k=x, v=x, block_tables=tables, context_lengths=lengths,
              cu_seqlens_q=cu, max_seqlen_q=3, key_scale=s, value_scale=t)
    pkg.append_kv(**ok)
    f, f2 = (torch.zeros(4, 16, 2, 64, device=dev).to(FP8) for _ in range(2))
    per = torch.ones(4, 16, 2, device=dev)
    for bad in (dict(key_scale=None, value_scale=None), dict(value_scale=None), dict(value_cache=k),
                dict(value_scale=s), dict(key_scale=per, value_scale=per.clone()),
                dict(key_scale=torch.tensor(1.0, device=dev), value_scale=torch.tensor(1.0, device=dev)),
                dict(key_cache=f, value_cache=f2, key_scale=per[:3], value_scale=per[:3].clone()),
                dict(key_cache=f, value_cache=f2, key_scale=s.half(), value_scale=t.half()),
                dict(key_cache=x.new_zeros(4, 16, 2, 64), value_cache=x.new_zeros(4, 16, 2, 64)),
                dict(key_cache=k.float(), value_cache=v.float(), key_scale=None, value_scale=None),
                dict(k=x[:2]), dict(v=x.float()), dict(k=x[..., :32], v=x[..., :32]), dict(k=x[:, :1], v=x[:, :1]),
                dict(key_scale=s[:3], value_scale=t[:3]), dict(cu_seqlens_q=cu[:1]), dict(max_seqlen_q=-1),
                dict(context_lengths=lengths.cpu()), dict(q=x[:2]), dict(q=x.float()),
                dict(positions=torch.zeros(2, dtype=torch.long, device=dev)),
                dict(rotary=pkg.Rotary(66, device=dev)),
                dict(key_cache=k[:1].expand(4, 16, 2, 64), value_cache=v[:1].expand(4, 16, 2, 64)),
                dict(key_cache=k.long(), value_cache=v.long())):
        with pytest.raises(ValueError):
            pkg.append_kv(**{**ok, **bad})
    ok = dict(key_cache=k, value_cache=v, block_tables=tables, context_lengths=lengths, cu_seqlens=cu,
              max_seqlen=3, rows=3, key_scale=s, value_scale=t)
    for bad in (dict(key_scale=None, value_scale=None), dict(rows=-1), dict(dtype=torch.int8),
                dict(key_scale=per, value_scale=per), dict(cu_seqlens=cu[:1]), dict(max_seqlen=-1)):
        with pytest.raises(ValueError):
            pkg.load_kv(**{**ok, **bad})
