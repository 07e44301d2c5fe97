"""Attention over block-scaled pools whose scales differ widely from block to block, against float64
(``Case`` and its tolerance: ``test_gpu_block_attention``)."""

import pytest
import torch

from tests.test_gpu_block_attention import CODES, Case, _near, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kernel(pkg):
    return pkg.MI355XPagedAttention()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,dim,bs", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32), (torch.bfloat16, 96, 64),
                                          (torch.float16, 128, 48), (torch.bfloat16, 128, 8)])
def test_prompts_whose_key_scales_differ_by_tile(kernel, dev, codes, dtype, dim, bs):
    """Key scales a hundredfold apart, so that a tile's weights by another tile's scales would show; every
    repetition has the same bits, whatever its waves wait for."""
    _say("key scales", codes, dtype, dim, bs)
    c = Case(codes, dtype, [(1100, 1100), (900, 200), (130, 129), (65, 65), (64, 64)], 4, 2, dim, bs, seed=21,
             spread=0.01)
    for window in (0, 300):
        got = c.packed(kernel, dev, window)
        _near(got, *c.expect(window), c.q)
        for _ in range(8):
            assert torch.equal(c.packed(kernel, dev, window), got)


def _single(kernel, dev, c, window=0, lengths=None):
    """The rows of a packed case one by one; by their own lengths where those are given."""
    q, k, v, tables, _, _, ks, vs = c.args(dev)
    seq = torch.cat([torch.full((n,), s) for s, (_, n) in enumerate(c.seqs)]).to(dev)
    if lengths is None:
        lengths = torch.cat([torch.arange(n - r + 1, n + 1) for n, r in c.seqs])
    rest = (tables[seq], lengths.int().to(dev))
    if window:
        return kernel.windowed(q, k[:, 1], v[:, 1], *rest, window, ks[:, 1], vs[:, 1]).cpu()
    return kernel(q, k[:, 1], v[:, 1], *rest, ks[:, 1], vs[:, 1]).cpu()


ACROSS = [(706, 5), (690, 4), (1025, 5), (33, 20), (20, 20), (1030, 16), (1281, 3), (17, 2)]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,hq,hkv,dim,bs", [(torch.bfloat16, 8, 4, 128, 16), (torch.float16, 4, 1, 64, 16),
                                                 (torch.bfloat16, 2, 2, 256, 32), (torch.bfloat16, 8, 4, 96, 16)])
@pytest.mark.parametrize("log2", (12, 24, 40, 90))
def test_rows_beside_a_block_of_larger_values(pkg, kernel, dev, codes, dtype, hq, hkv, dim, bs, log2):
    """The scale of a block that only the rows beside it see does not reach a row: packed rows have the bits
    of single ones, and are as near float64 as without it."""
    if dtype == torch.float16 and log2 > 12:
        return  # (such outputs are past its largest number)
    _say("larger beside", codes, dtype, dim, log2)
    c = Case(codes, dtype, ACROSS, hq, hkv, dim, bs, seed=22)
    last = torch.tensor([int(c.tables[s][-(-n // bs) - 1]) for s, (n, _) in enumerate(c.seqs)])
    c.vs[last] *= 2.0 ** log2
    c.q *= 2  # (weights over a wider range)
    got = c.packed(kernel, dev)
    assert torch.equal(got, _single(kernel, dev, c))
    assert torch.equal(c.packed(pkg.MI355XPagedAttention(compensate=True), dev),
                       _single(pkg.MI355XPagedAttention(compensate=True), dev, c))
    want, most = c.expect()
    reads = torch.cat([torch.arange(n - r, n) // bs == (n - 1) // bs for n, r in c.seqs])
    _near(got[~reads], want[~reads], most[~reads], c.q)
    if log2 <= 12:
        _near(got, want, most, c.q)
    # a sliding window that the first rows' larger block leaves
    first = torch.tensor([int(c.tables[s][(n - r - 32) // bs]) for s, (n, r) in enumerate(c.seqs) if n - r > 48])
    c.vs[first] *= 2.0 ** min(log2, 24)
    assert torch.equal(c.packed(kernel, dev, window=33), _single(kernel, dev, c, window=33))


@pytest.mark.parametrize("codes", CODES)
def test_row_lengths_far_apart_beside_larger_values(kernel, dev, codes):
    """Explicit row lengths in any order, every block with values a thousand times those of the one before."""
    _say("lengths apart", codes)
    c = Case(codes, torch.bfloat16, [(900, 30), (130, 14)], 4, 2, 128, 16, seed=23)
    for s, (n, _) in enumerate(c.seqs):
        for i in range(-(-n // 16)):
            c.vs[int(c.tables[s][i])] *= 2.0 ** (10 * (i % 9))
    g = torch.Generator().manual_seed(24)
    rl = torch.cat([torch.randint(0, n + 1, (r,), generator=g) for n, r in c.seqs]).int()
    q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
    got = kernel.prefill(q, k[:, 1], v[:, 1], tables, lengths, cu, 30, ks[:, 1], vs[:, 1], row_lengths=rl.to(dev))
    assert torch.equal(got.cpu(), _single(kernel, dev, c, lengths=rl))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,hq,hkv,dim,bs", [(torch.bfloat16, 8, 2, 128, 16), (torch.bfloat16, 4, 4, 64, 64),
                                                 (torch.bfloat16, 2, 1, 96, 8), (torch.float16, 4, 4, 128, 32)])
@pytest.mark.parametrize("log2", (12, 30, 75))
def test_prompts_beside_a_block_of_larger_values(kernel, dev, codes, dtype, hq, hkv, dim, bs, log2):
    """Rows of a prompt whose last block's values are far larger: those that do not see it are as near float64
    as without it; so are rows that a sliding window took past one."""
    if dtype == torch.float16 and log2 > 12:
        return  # (such outputs are past its largest number)
    _say("prompts, larger beside", codes, dtype, dim, bs, log2)
    c = Case(codes, dtype, [(400, 400), (333, 100), (129, 129), (70, 65)], hq, hkv, dim, bs, seed=25)
    last = torch.tensor([int(c.tables[s][-(-n // bs) - 1]) for s, (n, _) in enumerate(c.seqs)])
    c.vs[last] *= 2.0 ** log2
    got = c.packed(kernel, dev)
    want, most = c.expect()
    reads = torch.cat([torch.arange(n - r, n) // bs == (n - 1) // bs for n, r in c.seqs])
    _near(got[~reads], want[~reads], most[~reads], c.q)
    if log2 <= 12:
        _near(got, want, most, c.q)
    c.vs[last] *= 2.0 ** -log2
    c.vs[int(c.tables[0][300 // bs])] *= 2.0 ** log2
    got, (want, most) = c.packed(kernel, dev, 50), c.expect(50)
    at = torch.cat([torch.arange(n - r, n) for n, r in c.seqs])
    reads = (at < 400) & (torch.arange(len(at)) < 400) & (at // bs >= 300 // bs) & ((at - 49) // bs <= 300 // bs)
    _near(got[~reads], want[~reads], most[~reads], c.q)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,dim,bs", [(4, 2, 128, 8), (8, 1, 64, 24), (2, 2, 256, 3), (6, 2, 96, 40)])
@pytest.mark.parametrize("factor", (1e-2, 1e-3, 300.0))
def test_small_and_large_values_in_blocks_of_any_size(kernel, dev, codes, hq, hkv, dim, bs, factor):
    """fp16 weights keep their bits where blocks hold no whole 16-position tiles, whatever the size of the
    values and beside a block of larger ones; packed rows have the bits of single ones."""
    _say("any block", codes, dim, bs, factor)
    c = Case(codes, torch.float16, ACROSS, hq, hkv, dim, bs, seed=26, spread=0.05)
    c.vs *= factor
    got = c.packed(kernel, dev)
    _near(got, *c.expect(), c.q)
    assert torch.equal(got, _single(kernel, dev, c))
    last = torch.tensor([int(c.tables[s][-(-n // bs) - 1]) for s, (n, _) in enumerate(c.seqs)])
    c.vs[last] *= 64 if factor > 1 else 2.0 ** 16
    got, (want, most) = c.packed(kernel, dev), c.expect()
    assert torch.equal(got, _single(kernel, dev, c))
    reads = torch.cat([torch.arange(n - r, n) // bs == (n - 1) // bs for n, r in c.seqs])
    _near(got[~reads], want[~reads], most[~reads], c.q)
    got = c.packed(kernel, dev, window=21)
    assert torch.equal(got, _single(kernel, dev, c, window=21))


def _bytes(x):
    return x.contiguous().view(torch.uint8)


def test_stores_are_refused_before_the_append(kernel, dev):
    """A call that the attention would refuse leaves the cache and its scales as they were."""
    _say("refused stores")
    c = Case(torch.int8, torch.bfloat16, [(10, 3)], 4, 2, 64, 16, seed=27)
    q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
    k, v, ks, vs = k[:, 1], v[:, 1], ks[:, 1], vs[:, 1]
    new = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=dev) * 50
    apart = torch.zeros(1, 2, dtype=torch.int32, device=dev)[:, ::2]  # (one column, two apart)
    before = [x.clone() for x in (k, v, ks, vs)]
    for bad in (dict(block_tables=apart), dict(q=q[:, :0]), dict(q=q[:, :3]), dict(max_seqlen_q=0),
                dict(max_seqlen_q=1 << 31)):
        args = dict(q=q, block_tables=tables, max_seqlen_q=3)
        args.update(bad)
        with pytest.raises(ValueError):
            kernel.prefill_store(args["q"], new, new, k, v, args["block_tables"], lengths, cu,
                                 args["max_seqlen_q"], ks, vs)
        torch.cuda.synchronize()
        for a, b in zip((k, v, ks, vs), before):
            assert torch.equal(_bytes(a), _bytes(b))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("rows", (3, 70))
def test_stores_by_a_bound_and_over_strides_of_8_bytes(kernel, dev, codes, rows):
    """``max_seqlen_q`` far above the windows, and 96-dim heads 104 bytes apart: the same outputs and scales."""
    _say("store bound", codes, rows)
    c = Case(codes, torch.bfloat16, [(rows + 9, rows)], 4, 2, 96, 16, seed=28)
    q, k, v, tables, lengths, cu, ks, vs = c.args(dev)
    g = torch.Generator().manual_seed(29)
    new_k, new_v = (torch.randn(rows, 2, 96, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))

    def pool(x, apart):
        out = torch.zeros(x.shape[0], 16, 2, apart, dtype=torch.uint8, device=dev)[..., :96]
        return out.copy_(x[:, 1].view(torch.uint8)).view(codes)

    outs = []
    for apart, bound in ((96, rows), (104, rows), (96, 2 ** 31 - 1), (104, 2 ** 31 - 1)):
        held = pool(k, apart), pool(v, apart), ks[:, 1].clone(), vs[:, 1].clone()
        out = kernel.prefill_store(q, new_k, new_v, *held[:2], tables, lengths, cu, bound, *held[2:])
        outs.append((out, *map(_bytes, held)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_calls_of_more_units_than_a_launch(kernel, dev):
    """2^24 units of 256 threads, nearly all without keys: single rows over tables padded to 65536 positions, and
    prompts whose longest window is known by its bound; as the same rows in a small call."""
    _say("past one launch")
    n, heads, width = 4112, 64, 4096  # 4112 x 64 x 64 chunks
    g = torch.Generator(device=dev).manual_seed(30)
    k, v = (torch.randint(-127, 128, (64, 16, heads, 64), generator=g, device=dev, dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.rand(64, heads, generator=g, device=dev) * 0.02 + 0.001 for _ in range(2))
    few = torch.randint(0, 64, (n, 4), generator=g, device=dev, dtype=torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    tables[:, :4] = few
    lengths = torch.randint(1, 65, (n,), generator=g, device=dev, dtype=torch.int32)
    q = torch.randn(n, heads, 64, generator=g, device=dev).to(torch.bfloat16)
    got = kernel(q, k, v, tables, lengths, ks, vs)
    for part in (slice(0, 40), slice(n // 2 - 20, n // 2 + 20), slice(n - 40, n)):
        assert torch.equal(got[part], kernel(q[part], k, v, few[part].contiguous(), lengths[part], ks, vs))
    del tables
    # 64 rows of every eighth sequence, none of the others: 1040 x 64 heads x 256 groups of 128 rows
    seqs, bound = 1040, 32768
    counts = torch.zeros(seqs, dtype=torch.int32, device=dev)
    counts[::8] = 64
    counts[-1] = 64
    cu = torch.cat([counts.new_zeros(1), counts.cumsum(0).int()])
    rows = int(cu[-1])
    q = torch.randn(rows, heads, 64, generator=g, device=dev).to(torch.bfloat16)
    args = (few[:seqs].contiguous(), counts, cu)
    got = kernel.prefill(q, k, v, *args, bound, ks, vs)
    assert torch.equal(got, kernel.prefill(q, k, v, *args, 64, ks, vs))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,dim,bs", [(4, 2, 128, 8), (8, 1, 64, 24), (2, 2, 256, 3), (6, 2, 96, 40),
                                           (4, 2, 128, 16), (6, 2, 96, 32)])
def test_weights_are_rounded_to_fp16_whatever_the_queries(kernel, dev, codes, hq, hkv, dim, bs):
    """bfloat16 windows in blocks of any size.  A weight times its scale is float32 until it is rounded to fp16
    (2^-11, half a step), float32 scores put a weight off by 2^-18 and sums by 2^-16 over these lengths, and the
    output is rounded once (2^-8)."""
    _say("fp16 weights", codes, dim, bs)
    short = [(n, min(n, 5)) for n in range(1, 40)]
    c = Case(codes, torch.bfloat16, ACROSS + short, hq, hkv, dim, bs, seed=31)
    scales = c.vs.clone()
    for factor in (1.0, 2.0 ** -85, 2.0 ** 75):
        c.vs = scales * factor
        got, (want, most) = c.packed(kernel, dev), c.expect()
        near = most * (2.0 ** -11 + 2.0 ** -15) + want.abs() * 2.0 ** -8
        assert ((got.double() - want).abs() <= near * 1.01).all()
        assert torch.equal(got, _single(kernel, dev, c))
