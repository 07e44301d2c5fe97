"""Attention over 8-bit pools with one scale per block of tokens and kv head, against the same
attention in float64 over the numbers that the codes stand for."""

import math

import pytest
import torch

from oracle import rotary as orot

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
CODES = (FP8, torch.int8)


def _say(*args):
    print("[case]", *args, flush=True)


@pytest.fixture(scope="module")
def kernel(pkg):
    return pkg.MI355XPagedAttention()


class Case:
    def __init__(self, codes, dtype, seqs, hq, hkv, dim, bs, seed=0, spread=0.3):
        """``seqs``: (positions, q rows) per sequence; ``spread``: scales between it and 1."""
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.codes = seqs, codes
        need = [max(1, -(-n // bs)) for n, _ in seqs]
        blocks = sum(need) + 2
        shape = (blocks, 2, bs, hkv, dim)
        self.k, self.v = (torch.randint(-127, 128, shape, generator=g).to(torch.int8) if codes == torch.int8
                          else (torch.randn(shape, generator=g) * 90).clamp(-448, 448).to(FP8)
                          for _ in range(2))
        top = 127 if codes == torch.int8 else 300
        self.ks, self.vs = ((spread ** torch.rand(blocks, 2, hkv, generator=g)) * 2.5 / top
                            for _ in range(2))
        order = torch.randperm(blocks, generator=g).tolist()
        self.tables = torch.full((len(seqs), max(need)), -1, dtype=torch.int32)
        for s, n in enumerate(need):
            self.tables[s, :n] = torch.tensor([order.pop() for _ in range(n)])
        rows = sum(c for _, c in seqs)
        self.q = (torch.randn(rows, hq, dim, generator=g)).to(dtype)
        self.lengths = torch.tensor([n for n, _ in seqs], dtype=torch.int32)
        self.cu = torch.tensor([0, *torch.tensor([c for _, c in seqs]).cumsum(0).tolist()], dtype=torch.int32)
        self.most = max(c for _, c in seqs)

    def args(self, dev):
        return [x.to(dev) for x in (self.q, self.k, self.v, self.tables, self.lengths, self.cu, self.ks, self.vs)]

    def packed(self, kernel, dev, window=0):
        q, k, v, tables, lengths, cu, ks, vs = self.args(dev)
        return kernel.prefill(q, k[:, 1], v[:, 1], tables, lengths, cu, self.most, ks[:, 1], vs[:, 1],
                              window=window).cpu()

    def expect(self, window=0):
        """(attention in float64, the largest |value| that each output is a mean of)."""
        k, v = (orot.dequantized(c[:, 1], s[:, 1]) for c, s in ((self.k, self.ks), (self.v, self.vs)))
        group = self.q.shape[1] // self.k.shape[3]
        out, most = [], []
        for s, (n, c) in enumerate(self.seqs):
            blocks = self.tables[s][:max(1, -(-n // self.k.shape[2]))].long()
            kk, vv = (x[blocks].flatten(0, 1)[:n].repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
            q = self.q[self.cu[s]:self.cu[s + 1]].double().transpose(0, 1)
            x = q @ kk.transpose(1, 2) / math.sqrt(q.shape[-1])
            end = torch.arange(n - c + 1, n + 1)[:, None]
            at = torch.arange(n)[None]
            hidden = (at >= end) | ((at < end - window) if window else (at < 0))
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1).nan_to_num()
            out.append((p @ vv).transpose(0, 1))
            most.append((p @ vv.abs()).transpose(0, 1))
        return torch.cat(out), torch.cat(most)


def _near(got, want, most, q):
    """A weight is rounded to q's type before its product and once more by its value scale (float32), so an
    output is off by eps / 2 of its mean of |values|; float32 scores of magnitude up to 60 put a weight off by
    2^-18 (exponents), sums and the accumulators by 2^-16 over these lengths; the output is rounded once, below
    the smallest normal number by half a subnormal step (fp16: 2^-25, which is 1% of an output of 3e-6)."""
    info = torch.finfo(got.dtype)
    eps = info.eps if got.dtype != torch.float32 else 0.0
    near = most * (eps / 2 + 2.0 ** -15) + want.abs() * eps / 2 + info.smallest_normal * info.eps / 2
    assert got.isfinite().all()
    assert ((got.double() - want).abs() <= near * 1.01).all()


WINDOWS = [(1, 1), (5, 5), (16, 3), (17, 1), (700, 5), (1023, 4), (1024, 1), (1025, 5), (2200, 2), (3, 3)]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("hq,hkv,dim,bs", [(16, 4, 128, 16), (8, 8, 64, 16), (6, 2, 96, 32), (4, 2, 256, 16),
                                           (16, 4, 128, 8), (4, 2, 96, 24), (2, 1, 64, 3), (5, 5, 96, 48),
                                           (8, 1, 128, 64)])
def test_verify_windows(kernel, dev, codes, dtype, hq, hkv, dim, bs):
    """Windows over prefixes that end in every part of a block, a tile and a chunk; blocks of any size."""
    _say("block verify", codes, dtype, hq, hkv, dim, bs)
    c = Case(codes, dtype, WINDOWS, hq, hkv, dim, bs, seed=bs + dim)
    got = c.packed(kernel, dev)
    _near(got, *c.expect(), c.q)
    got = c.packed(kernel, dev, window=100)
    _near(got, *c.expect(100), c.q)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,hq,hkv,dim,bs", [(torch.float32, 4, 2, 128, 16), (torch.float32, 2, 1, 64, 8),
                                                 (torch.bfloat16, 4, 2, 32, 16), (torch.float16, 3, 3, 7, 5)])
def test_vector_form(kernel, dev, codes, dtype, hq, hkv, dim, bs):
    """float32 queries and head sizes that the matrix instructions do not serve."""
    _say("block vector", codes, dtype, dim, bs)
    c = Case(codes, dtype, [(1, 1), (40, 5), (700, 3), (1500, 2)], hq, hkv, dim, bs, seed=3)
    _near(c.packed(kernel, dev), *c.expect(), c.q)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,dim,bs", [(torch.bfloat16, 128, 16), (torch.float16, 128, 32), (torch.bfloat16, 96, 8),
                                          (torch.float16, 64, 16), (torch.bfloat16, 256, 16), (torch.float16, 96, 16),
                                          (torch.bfloat16, 64, 40)])
def test_prompts(kernel, dev, codes, dtype, dim, bs):
    """Long windows: prompts, chunks behind a prefix, ragged ones, with and without a sliding window."""
    _say("block prompts", codes, dtype, dim, bs)
    c = Case(codes, dtype, [(500, 500), (900, 200), (130, 129), (64, 64), (300, 1), (65, 65)], 4, 2, dim, bs, seed=4)
    for window in (0, 150):
        _near(c.packed(kernel, dev, window), *c.expect(window), c.q)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_single_rows_equal_packed_rows(kernel, dev, codes, dtype):
    """The per-row form, windows of a batch and the same windows alone: the same bits."""
    _say("block bitwise", codes, dtype)
    c = Case(codes, dtype, WINDOWS, 8, 4, 128, 16, seed=5)
    packed = c.packed(kernel, dev)
    q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
    seq = torch.cat([torch.full((n,), s) for s, (_, n) in enumerate(WINDOWS)])
    rows = torch.cat([torch.arange(n - r + 1, n + 1) for n, r in WINDOWS]).int()
    got = kernel(q, k[:, 1], v[:, 1], tables[seq.to(dev)], rows.to(dev), ks[:, 1], vs[:, 1]).cpu()
    assert torch.equal(got, packed)
    got = kernel.windowed(q, k[:, 1], v[:, 1], tables[seq.to(dev)], rows.to(dev), 33, ks[:, 1], vs[:, 1]).cpu()
    assert torch.equal(got, c.packed(kernel, dev, window=33))
    for s in (4, 8):
        a, b = int(c.cu[s]), int(c.cu[s + 1])
        alone = kernel.prefill(q[a:b], k[:, 1], v[:, 1], tables[s:s + 1], lengths[s:s + 1],
                               torch.tensor([0, b - a], dtype=torch.int32, device=dev), b - a, ks[:, 1], vs[:, 1])
        assert torch.equal(alone.cpu(), packed[a:b])


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("rows", (2, 80))
def test_scales_far_apart(kernel, dev, codes, rows):
    """Scales over six orders of magnitude, and small ones: fp16 weights lose nothing to them."""
    _say("block scales", codes, rows)
    for dtype in (torch.float16, torch.bfloat16):
        c = Case(codes, dtype, [(1400, rows), (90, rows)], 4, 2, 128, 16, seed=6, spread=1e-6)
        c.ks.fill_(2.5 / (127 if codes == torch.int8 else 300))
        _near(c.packed(kernel, dev), *c.expect(), c.q)
        c.vs *= 1e-3
        _near(c.packed(kernel, dev), *c.expect(), c.q)


@pytest.mark.parametrize("codes", CODES)
def test_empty_and_strange_rows(kernel, dev, codes):
    """No keys at all gives zeros; scales of 0 give the mean of zeros; what lies behind a sequence's end, its
    codes and other blocks' scales, has no effect; table entries outside the pool read block 0."""
    _say("block empty", codes)
    for rows in (3, 70):
        c = Case(codes, torch.bfloat16, [(0, rows), (rows, rows), (1, rows)], 4, 2, 64, 16, seed=7)
        got = c.packed(kernel, dev)
        assert not got[:rows].any() and not got[2 * rows:3 * rows - 1].any()
        b = Case(codes, torch.bfloat16, [(rows + 30, rows)], 4, 2, 64, 16, seed=8)
        before = b.packed(kernel, dev)
        used = b.tables[0].long()
        tail = (rows + 30) % 16
        if tail:
            if codes == FP8:
                b.k.view(torch.uint8)[used[-1], :, tail:] = 0x7F
                b.v.view(torch.uint8)[used[-1], :, tail:] = 0x7F
            else:
                b.k[used[-1], :, tail:] = -128
                b.v[used[-1], :, tail:] = -128
        others = torch.ones(b.k.shape[0], dtype=torch.bool)
        others[used] = False
        b.ks[others] = b.vs[others] = float("nan")
        assert torch.equal(b.packed(kernel, dev), before)
        b.vs[used] = 0.0
        assert not b.packed(kernel, dev).any()


@pytest.mark.parametrize("codes", CODES)
def test_row_lengths_and_compensated(pkg, kernel, dev, codes):
    """Explicit row lengths in any order equal the rows alone; the compensated product's outputs are no further
    off float64 than the plain one's."""
    _say("block rows", codes)
    c = Case(codes, torch.bfloat16, [(900, 4), (60, 4)], 8, 4, 128, 16, seed=9)
    q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
    rl = torch.tensor([900, 17, 500, 33, 1, 60, 16, 5], dtype=torch.int32, device=dev)
    got = kernel.prefill(q, k[:, 1], v[:, 1], tables, lengths, cu, 4, ks[:, 1], vs[:, 1], row_lengths=rl)
    seq = torch.tensor([0] * 4 + [1] * 4, device=dev)
    assert torch.equal(got, kernel(q, k[:, 1], v[:, 1], tables[seq], rl, ks[:, 1], vs[:, 1]))
    want, most = c.expect()
    plain = c.packed(kernel, dev)
    better = c.packed(pkg.MI355XPagedAttention(compensate=True), dev)
    _near(better, want, most, c.q)
    assert (better.double() - want).norm() <= (plain.double() - want).norm()


@pytest.mark.parametrize("codes", CODES)
def test_far_blocks(kernel, dev, codes):
    """Offsets past 32 bits: the last blocks of a pool of more than 2^32 codes."""
    _say("block far", codes)
    bs, hkv, dim = 64, 8, 128
    blocks = (1 << 32) // (bs * hkv * dim) + 40
    raw_k, raw_v = (torch.zeros(blocks, bs, hkv, dim, dtype=torch.uint8, device=dev) for _ in range(2))
    c = Case(codes, torch.bfloat16, [(150, 5)], 8, hkv, dim, bs, seed=10)
    n = c.k.shape[0]
    raw_k[-n:] = c.k[:, 1].contiguous().view(torch.uint8).to(dev)
    raw_v[-n:] = c.v[:, 1].contiguous().view(torch.uint8).to(dev)
    ks, vs = (torch.zeros(blocks, hkv, device=dev) for _ in range(2))
    ks[-n:], vs[-n:] = c.ks[:, 1].to(dev), c.vs[:, 1].to(dev)
    got = kernel.prefill(c.q.to(dev), raw_k.view(codes), raw_v.view(codes), c.tables.to(dev) + (blocks - n),
                         c.lengths.to(dev), c.cu.to(dev), 5, ks, vs)
    _near(got.cpu(), *c.expect(), c.q)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("rows", (5, 70))
def test_a_layer_step_by_step(pkg, dev, codes, rows):
    """What a layer does, over several steps of several requests: keys rotated and appended, then attention with
    the rotated queries; the same through ``prefill_store`` with rows rotated before; captured and replayed."""
    _say("layer", codes, rows)
    backend = pkg.create_backend("auto", dev, torch.bfloat16, 64, 16)
    plan = pkg.Rotary(64, device=dev)
    g = torch.Generator().manual_seed(11)
    width = -(-4 * rows // 16) + 1
    made = []
    for _ in range(2):
        k, v = (torch.zeros(2 * width, 2, 16, 2, 64, dtype=torch.uint8, device=dev).view(codes) for _ in range(2))
        made.append((k[:, 1], v[:, 1], *(torch.zeros(2 * width, 2, 2, device=dev)[:, 1] for _ in range(2))))
    tables = torch.randperm(2 * width, generator=g).int().view(2, width).to(dev)
    cu = torch.tensor([0, rows, 2 * rows - 1], dtype=torch.int32, device=dev)
    total = 2 * rows - 1
    lengths = torch.zeros(2, dtype=torch.int32, device=dev)
    q, k, v = (torch.zeros(total, h, 64, dtype=torch.bfloat16, device=dev) for h in (4, 2, 2))

    def step(kc, vc, ks, vs):
        turned = pkg.append_kv(kc, vc, k, v, tables, lengths, cu, rows, ks, vs, rotary=plan, q=q)
        return backend.prefill(turned, kc, vc, tables, lengths, cu, rows, ks, vs)

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        step(*(x.clone() for x in made[0]))
    warm.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*made[0])
    keys, values = [[], []], [[], []]
    for i in range(4):
        new = torch.tensor([(i + 1) * rows, (i + 1) * (rows - 1)], dtype=torch.int32)
        lengths.copy_(new)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        assert torch.equal(out, step(*made[1]))
        for a, b in zip(*made):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        # against the rows kept as they were: a cached number is off by half a step of its code (and of every
        # larger scale that its block took, at most 15 of them), 2^-4 or 1 / 254 of the block's largest
        turns = plan.turns.cpu()
        for s, (n, c) in enumerate(zip(new.tolist(), (rows, rows - 1))):
            a, b = int(cu[s]), int(cu[s + 1])
            at = torch.arange(n - c, n)
            keys[s].append(orot.rotate(k[a:b].cpu(), at, turns))
            values[s].append(v[a:b].cpu().double())
            kk, vv = (torch.cat(x[s]).repeat_interleave(2, 1).transpose(0, 1) for x in (keys, values))
            x = orot.rotate(q[a:b].cpu(), at, turns).transpose(0, 1) @ kk.transpose(1, 2) / 8
            p = torch.softmax(x.masked_fill(torch.arange(n)[None] > at[:, None], -math.inf), -1)
            want = (p @ vv).transpose(0, 1)
            off = (out[a:b].cpu().double() - want).norm() / want.norm()
            # int8 1 / 254 of amax (about 3.5 for N(0, 1)), uniform: rms 0.008 a number; e4m3 rms 2^-4 / sqrt 3
            # = 0.036; keys move a score by that over 1 and so weights by it, values directly; doubled twice for
            # the rounding again of codes
            assert off < 4 * (0.008 if codes == torch.int8 else 0.036) * 2
    # the store in one call, on a third cache
    third = [torch.zeros_like(x) for x in made[0]]
    lengths.copy_(torch.tensor([rows, rows - 1]))
    at = torch.cat([torch.arange(rows), torch.arange(rows - 1)]).to(dev)
    got = backend.prefill_store(q, k, v, third[0], third[1], tables, lengths, cu, rows, third[2], third[3])
    fourth = [torch.zeros_like(x) for x in made[0]]
    pkg.append_kv(fourth[0], fourth[1], k, v, tables, lengths, cu, rows, fourth[2], fourth[3])
    assert torch.equal(got, backend.prefill(q, fourth[0], fourth[1], tables, lengths, cu, rows, fourth[2], fourth[3]))
    for a, b in zip(third, fourth):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("codes", CODES)
def test_queries_that_are_not_numbers(kernel, dev, codes):
    """A NaN query gives NaN, in its own row alone; a sequence's blocks before a sliding window may hold any
    scales (where blocks hold whole tiles, and in prompts)."""
    _say("block nan")
    for rows in (4, 70):
        for bs in (16, 8):
            c = Case(codes, torch.bfloat16, [(1500, rows), (90, rows)], 4, 2, 64, bs, seed=14)
            want = c.packed(kernel, dev)
            c.q[1, 2], c.q[rows + 2, 1, 5] = float("nan"), float("nan")
            got = c.packed(kernel, dev)
            bad = torch.zeros(got.shape[:2], dtype=torch.bool)
            bad[1, 2] = bad[rows + 2, 1] = True
            assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])
            c = Case(codes, torch.bfloat16, [(1500, rows)], 4, 2, 64, bs, seed=15)
            want = c.packed(kernel, dev, window=40)
            hidden = c.tables[0][:(1500 - rows + 1 - 40) // bs].long()
            c.ks[hidden] = c.vs[hidden] = float("nan")
            if bs == 16 or rows == 70:
                assert torch.equal(c.packed(kernel, dev, window=40), want)


def test_a_batch_with_padding(kernel, dev):
    """Sequences without rows or without keys between others, and rows behind the last sequence: these are left."""
    _say("block padding")
    for codes in CODES:
        c = Case(codes, torch.bfloat16, [(700, 3), (0, 2), (1100, 0), (33, 1), (0, 0)], 4, 2, 64, 16, seed=16)
        q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
        got = c.packed(kernel, dev)
        for s in (0, 3):
            a, b = int(c.cu[s]), int(c.cu[s + 1])
            one = kernel.prefill(q[a:b], k[:, 1], v[:, 1], tables[s:s + 1], lengths[s:s + 1],
                                 torch.tensor([0, b - a], dtype=torch.int32, device=dev), b - a, ks[:, 1], vs[:, 1])
            assert torch.equal(one.cpu(), got[a:b])
        assert not got[3:5].any()


def test_tables_without_columns(kernel, dev):
    """No sequence has a block: rows of zeros, whatever the lengths."""
    _say("block no columns")
    for codes in CODES:
        for rows in (1, 5, 80):
            c = Case(codes, torch.bfloat16, [(90, rows), (90, rows)], 4, 2, 64, 16, seed=17)
            c.tables = c.tables[:, :0].contiguous()
            assert not c.packed(kernel, dev).any()


def test_more_pairs_than_a_workgroup_lists(kernel, dev):
    """Batches past the persistent kernel's index run one workgroup per unit: the same bits."""
    _say("block many")
    for codes in CODES:
        c = Case(codes, torch.bfloat16, [(40, 1)], 2, 1, 64, 16, seed=12)
        q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
        n = 8200
        got = kernel(q.expand(n, -1, -1).contiguous(), k[:, 1], v[:, 1], tables.expand(n, -1).contiguous(),
                     lengths.expand(n).contiguous(), ks[:, 1], vs[:, 1])
        one = kernel(q, k[:, 1], v[:, 1], tables, lengths, ks[:, 1], vs[:, 1])
        assert torch.equal(got, one.expand(n, -1, -1))


def test_refusals(pkg, kernel, dev):
    c = Case(torch.int8, torch.bfloat16, [(40, 2)], 4, 2, 64, 16, seed=13)
    q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
    k, v, ks, vs = k[:, 1], v[:, 1], ks[:, 1], vs[:, 1]
    kernel.prefill(q, k, v, tables, lengths, cu, 2, ks, vs)
    one = torch.tensor(1.0, device=dev)
    per = torch.ones(k.shape[:3], device=dev)
    for a, b in ((None, None), (one, one), (per, per), (ks, None), (ks[:3], vs[:3]), (ks, vs.contiguous()),
                 (ks.half(), vs.half()), (ks[:, :1], vs[:, :1])):
        with pytest.raises(ValueError):
            kernel.prefill(q, k, v, tables, lengths, cu, 2, a, b)
    half = torch.zeros(k.shape, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        kernel.prefill(q, half, half.clone(), tables, lengths, cu, 2, ks, vs)
    words = torch.ones(2, 1, dtype=torch.int64, device=dev)
    for x, y in ((k, v), (half.to(FP8), half.to(FP8))):
        with pytest.raises((ValueError, RuntimeError)):
            kernel.tree(q, x, y, tables, lengths, cu, 2, words, ks, vs)
    with pytest.raises(ValueError):
        kernel.prefill_store(q, q[:, :2], q[:, :2], k, v, tables, lengths, cu, 2, ks, vs,
                             row_lengths=torch.tensor([3, 4], dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        pkg.store_kv(k, v, k[0, :2], v[0, :2], torch.zeros(2, dtype=torch.long, device=dev),
                     torch.zeros(2, dtype=torch.long, device=dev))
