"""Tree attention on the GPU against plain float64 attention over the visible positions."""

import math

import pytest
import torch

from tests.tree_cases import FP8, make_case, reference

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def call(pkg, dev, c, window=0, **over):
    kernel = pkg.create_backend("auto", dev, c.q.dtype, c.q.shape[-1], c.block)
    a = dict(q=c.q, key_cache=c.k, value_cache=c.v, block_tables=c.tables,
             context_lengths=c.lengths, cu_seqlens_q=c.cu, tree_mask=c.mask, key_scale=c.k_scale,
             value_scale=c.v_scale)
    a.update(over)
    a = {k: (v.to(dev) if torch.is_tensor(v) and v.device.type == "cpu" else v)
         for k, v in a.items()}
    return kernel.tree(max_seqlen_q=over.get("max_seqlen_q", c.max_q), window=window,
                       **{k: v for k, v in a.items() if k != "max_seqlen_q"})


def check(got, c, window=0, rows=None, fine=False):
    want, tol = reference(c, window, fine)
    got = got.double().cpu()
    if rows is not None:
        got, want, tol = got[rows], want[rows], tol[rows]
    assert torch.isfinite(got).all()
    over = (got - want).abs() - tol
    assert over.max() <= 0, f"{float(over.max())} beyond the tolerance"


# (nodes, ctx, q heads, kv heads, dim, type, kv, block size, window)
SHAPES = [
    # one row block of each width, 16-bit pools
    ([1], [1], 1, 1, 128, BF, "same", 16, 0),
    ([1, 5], [700, 33], 4, 4, 128, BF, "same", 16, 0),
    ([16, 3, 32], [515, 64, 32], 2, 2, 64, HF, "same", 16, 0),
    ([16, 16], [300, 1025], 8, 2, 128, BF, "same", 16, 0),       # 64 rows
    ([26, 9, 31], [260, 511, 640], 16, 4, 128, BF, "same", 16, 0),  # 124 rows
    ([26, 9], [260, 511], 16, 4, 64, HF, "same", 32, 0),
    ([33, 70], [129, 400], 8, 2, 128, HF, "same", 16, 0),        # three row blocks, two words
    ([12, 40], [100, 333], 5, 5, 96, BF, "same", 16, 0),
    ([64, 20], [200, 90], 3, 3, 96, HF, "same", 16, 0),
    ([40], [777], 6, 2, 96, BF, "same", 16, 0),
    ([9, 20], [257, 96], 2, 2, 256, BF, "same", 16, 0),
    ([40], [300], 4, 1, 256, HF, "same", 16, 0),
    # fp8 pools
    ([16, 7], [515, 96], 16, 8, 128, BF, "fp8", 16, 0),
    ([16, 7], [515, 96], 16, 8, 128, HF, "fp8_vector", 16, 0),
    ([30, 50], [515, 96], 8, 4, 128, BF, "fp8_vector", 16, 0),
    ([30, 50], [400, 96], 8, 2, 128, HF, "fp8", 16, 0),
    ([12, 31], [300, 77], 2, 2, 64, BF, "fp8", 16, 0),
    ([12, 31], [300, 77], 4, 2, 64, HF, "fp8_vector", 8, 0),
    ([50, 31], [300, 77], 4, 2, 64, BF, "fp8_vector", 16, 0),
    ([12, 31], [300, 77], 5, 5, 96, BF, "fp8", 16, 0),
    ([12, 40], [300, 77], 10, 5, 96, HF, "fp8_vector", 16, 0),
    ([44], [300], 10, 2, 96, BF, "fp8", 16, 0),
    ([12, 9], [300, 77], 2, 1, 256, BF, "fp8", 16, 0),
    ([30], [300], 4, 1, 256, HF, "fp8_vector", 16, 0),
    # block sizes
    ([16, 7], [515, 96], 4, 2, 128, BF, "same", 8, 0),
    ([16, 7], [515, 96], 4, 2, 128, BF, "fp8", 64, 0),
    ([16, 7], [200, 96], 4, 2, 128, BF, "same", 12, 0),          # vector form
    ([16, 7], [515, 96], 4, 2, 128, BF, "same", 24, 0),
    # sliding windows: in the prefix, inside the tree, one position
    ([16, 20], [515, 96], 4, 2, 128, BF, "same", 16, 100),
    ([40, 70], [515, 96], 4, 2, 128, BF, "fp8_vector", 16, 3),
    ([40, 9], [515, 9], 4, 4, 64, HF, "same", 16, 1),
    ([20], [300], 2, 2, 80, BF, "same", 16, 37),
    # the vector form: float32, other head sizes
    ([16, 7], [215, 96], 4, 2, 128, F32, "same", 16, 0),
    ([16, 7], [215, 96], 4, 2, 64, F32, "fp8_vector", 16, 50),
    ([9, 70], [50, 70], 2, 1, 7, BF, "same", 16, 0),
    ([9, 70], [50, 80], 2, 1, 80, HF, "fp8", 5, 0),
    # the largest tree; a tree that fills its cache
    ([256], [300], 2, 1, 64, BF, "same", 16, 0),
    ([200, 1], [200, 1], 4, 1, 128, BF, "same", 16, 0),
    ([130], [420], 2, 2, 64, BF, "same", 16, 60),
]


@pytest.mark.parametrize("nodes,ctx,hq,hkv,dim,dtype,kv,block,window", SHAPES)
def test_matches_plain_attention(pkg, dev, nodes, ctx, hq, hkv, dim, dtype, kv, block, window):
    c = make_case(nodes, ctx, hq, hkv, dim, dtype, kv, block, seed=sum(nodes) + dim)
    check(call(pkg, dev, c, window), c, window)


@pytest.mark.parametrize("dtype,kv,dim", [(BF, "same", 128), (HF, "fp8_vector", 64),
                                          (F32, "same", 32)])
def test_masks_that_are_no_trees(pkg, dev, dtype, kv, dim):
    """Any bits: rows that see nothing of the tree, only others, everything; bits past the tree."""
    g = torch.Generator().manual_seed(5)
    nodes, ctx = [20, 70, 5, 3], [20, 150, 5, 40]
    bits = []
    for m in nodes:
        rows = []
        for i in range(m):
            kind = int(torch.randint(0, 4, (), generator=g))
            noise = int(torch.randint(0, 1 << 30, (), generator=g)) << 75
            inside = {0: 0, 1: (1 << m) - 1, 2: 1 << ((i + 1) % m),
                      3: int(torch.randint(0, 1 << 20, (), generator=g)) % (1 << m)}[kind]
            rows.append(inside | (noise & ~((1 << m) - 1)) | (1 << 90))
        bits.append(rows)
    bits[2][1] = 1 << 90  # sees nothing: the tree fills its cache
    c = make_case(nodes, ctx, 4, 2, dim, dtype, kv, bits=bits, words=3)
    got = call(pkg, dev, c)
    check(got, c)
    assert (got[91] == 0).all()


@pytest.mark.parametrize("dtype,kv,dim,nodes", [
    (BF, "same", 128, [16, 9]), (HF, "same", 64, [30, 70]), (BF, "same", 96, [40, 9]),
    (BF, "fp8", 128, [16, 9]), (HF, "fp8_vector", 64, [50, 40]), (BF, "same", 256, [20, 9]),
    (F32, "same", 32, [16, 9]), (BF, "same", 80, [9, 3])])
@pytest.mark.parametrize("window", [0, 40])
def test_hidden_values_have_no_effect(pkg, dev, dtype, kv, dim, nodes, window):
    """NaN and infinities at positions that some rows do not see: those rows are unmoved, the
    rows that see them show them."""
    c = make_case(nodes, [200, 131], 4, 2, dim, dtype, kv, seed=3)
    clean, _ = reference(c, window)
    spoilt = {}
    from tests.tree_cases import visible
    for s in range(2):
        sees = visible(c, s, window)
        base = c.ctx[s] - c.nodes[s]
        # hidden from some rows, seen by at least itself: nodes 2 and the last; and the first
        # position that a sliding window takes from some rows only
        picks = [base + 2, c.ctx[s] - 1]
        if window:
            part = (sees.any(0) & ~sees.all(0))[:base].nonzero().flatten().tolist()
            picks += part[:1]
        for i, pos in enumerate(picks):
            blk, off = int(c.tables[s, pos // c.block]), pos % c.block
            bad = math.nan if kv != "same" or i % 2 else math.inf
            for pool, head in ((c.v, 0), (c.k, 1)):
                x = pool[blk, off].float()
                x[head, dim // 2] = bad
                pool[blk, off] = x.to(pool.dtype)
            if kv == "fp8_vector" and i == 1:
                c.v_scale[blk, off, 1] = math.nan
            spoilt.setdefault(s, []).append(pos)
    got = call(pkg, dev, c, window).double().cpu()
    _, tol = reference(c, window)
    begin = 0
    for s in range(2):
        sees = visible(c, s, window)
        hit = sees[:, spoilt[s]].any(1)
        assert hit.any() and not hit.all()
        rows = torch.arange(begin, begin + c.nodes[s])
        ok = rows[~hit]
        over = (got[ok] - clean[ok]).abs() - tol[ok]
        assert torch.isfinite(got[ok]).all() and over.max() <= 0
        # kv head 0: the value's dim only; kv head 1: a key spoils the whole row
        assert not torch.isfinite(got[rows[hit], 0, dim // 2]).any()
        rest = [d for d in range(dim) if d != dim // 2]
        assert torch.isfinite(got[rows[hit], 0][:, rest]).all()
        assert torch.isnan(got[rows[hit], 2]).any()
        begin += c.nodes[s]


@pytest.mark.parametrize("kv", ["same", "fp8"])
def test_long_contexts_split_over_workgroups(pkg, dev, kv):
    """Sequences far longer than a share, next to short ones and empty ones."""
    c = make_case([7, 0, 2, 26, 1], [9001, 0, 2, 4100, 3000], 4, 2, 128, BF, kv, seed=8)
    check(call(pkg, dev, c), c)


def test_more_sequences_than_threads(pkg, dev):
    """The shares of 600 sequences, some without rows or keys."""
    g = torch.Generator().manual_seed(1)
    nodes = [int(x) for x in torch.randint(0, 4, (600,), generator=g)]
    ctx = [m + int(x) for m, x in zip(nodes, torch.randint(0, 90, (600,), generator=g))]
    nodes[-1], ctx[-1] = 3, 50
    c = make_case(nodes, ctx, 2, 1, 64, BF, seed=2)
    check(call(pkg, dev, c), c)


def test_sequences_without_keys_give_zeros(pkg, dev):
    c = make_case([3, 2], [40, 20], 4, 2, 128, BF)
    got = call(pkg, dev, c, context_lengths=torch.tensor([0, -5], dtype=torch.int32))
    assert (got == 0).all()


def test_length_below_the_tree(pkg, dev):
    """Nodes before position 0 do not exist: the rest sees what is left."""
    c = make_case([10], [10], 2, 2, 64, BF, seed=4)
    got = call(pkg, dev, c, context_lengths=torch.tensor([6], dtype=torch.int32))
    c.ctx, c.lengths = [6], None
    # node j now lies at position j - 4
    import tests.tree_cases as tc
    sees = torch.zeros(10, 6, dtype=torch.bool)
    for i in range(10):
        for p in range(6):
            sees[i, p] = bool((c.bits[0][i] >> (p + 4)) & 1)
    old = tc.visible
    try:
        tc.visible = lambda *a: sees
        check(got, c)
    finally:
        tc.visible = old


def test_bad_lengths_and_table_entries_stay_inside_the_pool(pkg, dev):
    """A length past the table is cut to it; entries outside the pool read block 0."""
    c = make_case([4, 3], [100, 60], 2, 2, 128, BF, seed=6)
    c.k.nan_to_num_(0.0)
    c.v.nan_to_num_(0.0)
    tables = c.tables.clone()
    tables[0, 2], tables[1, 1] = -7, 1 << 30
    got = call(pkg, dev, c, block_tables=tables,
               context_lengths=torch.tensor([10 ** 6, 60], dtype=torch.int32))
    c.tables = tables.clone()
    c.tables[0, 2] = c.tables[1, 1] = 0
    c.ctx = [tables.shape[1] * c.block, 60]
    check(got, c)


def test_strided_queries_and_rows_past_the_sequences(pkg, dev):
    c = make_case([5, 9], [70, 130], 4, 2, 128, BF, seed=9)
    wide = torch.full((20, 6, 160), math.nan, dtype=BF)
    wide[:14, 1:5, 16:144] = c.q
    q = wide.to(dev)[:, 1:5, 16:144]
    mask = torch.full((20, 3), -1, dtype=torch.int64)
    mask[:14, :1] = c.mask
    got = call(pkg, dev, c, q=q, tree_mask=mask.to(dev)[:, :2])
    assert got.shape == (20, 4, 128)
    check(got[:14], c)


@pytest.mark.parametrize("shift", [1, 4])
def test_unaligned_views(pkg, dev, shift):
    """Pools and queries off the 16-byte pieces: the vector form."""
    c = make_case([5, 9], [70, 130], 4, 2, 64, HF, seed=9)

    def moved(x):
        flat = torch.empty(x.numel() + shift, dtype=x.dtype, device=dev)
        y = flat[shift:].view(x.shape)
        y.copy_(x)
        return y

    check(call(pkg, dev, c, key_cache=moved(c.k.contiguous()),
               value_cache=moved(c.v.contiguous()), q=moved(c.q)), c)


def test_offsets_past_32_bits(pkg, dev):
    """Blocks at the far end of a pool of more than 2^32 elements."""
    c = make_case([9], [150], 2, 2, 128, BF, seed=12)
    n = c.k.shape[0]
    far = (1 << 32) // (2 * 16 * 2 * 128) + 64
    pools = []
    for x in (c.k, c.v):
        big = torch.empty(far + n, 2, 16, 2, 128, dtype=BF, device=dev)
        big[far:, 1] = x.to(dev)
        pools.append(big[:, 1])
    got = call(pkg, dev, c, key_cache=pools[0], value_cache=pools[1],
               block_tables=c.tables + far)
    check(got, c)


def test_a_chain_equals_the_causal_window(pkg, dev):
    nodes, ctx = [5, 5, 3], [300, 1030, 77]
    c = make_case(nodes, ctx, 16, 4, 128, BF, seed=20,
                  bits=[[(2 << i) - 1 for i in range(m)] for m in nodes])
    got = call(pkg, dev, c)
    check(got, c)
    kernel = pkg.create_backend("auto", dev, BF, 128, 16)
    want = kernel.prefill(c.q.to(dev), c.k.to(dev), c.v.to(dev), c.tables.to(dev),
                          c.lengths.to(dev), c.cu.to(dev), 5)
    _, tol = reference(c)
    assert ((got.double() - want.double()).cpu().abs() <= 2 * tol).all()


def test_repeats_bit_for_bit_also_captured_and_on_another_stream(pkg, dev):
    c = make_case([26, 9], [2600, 511], 16, 4, 128, BF, seed=30)
    kernel = pkg.create_backend("auto", dev, BF, 128, 16)
    args = [x.to(dev) for x in (c.q, c.k, c.v, c.tables, c.lengths, c.cu)]
    mask = c.mask.to(dev)
    first = kernel.tree(*args, c.max_q, mask)
    check(first, c)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = kernel.tree(*args, c.max_q, mask)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = kernel.tree(*args, c.max_q, mask)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        out2 = kernel.tree(args[0] * 2, *args[1:], c.max_q, mask)
    doubled = kernel.tree(args[0] * 2, *args[1:], c.max_q, mask)
    for _ in range(3):
        out.zero_()
        out2.zero_()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(out2, doubled)
        junk = torch.randn(1 << 20, device=dev).sum().item()
        assert math.isfinite(junk)
    # new lengths in place: a replay follows the device's values
    args[4].copy_(torch.tensor([1500, 400], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    again = kernel.tree(*args, c.max_q, mask)
    assert torch.equal(out, again) and not torch.equal(again, first)
    assert torch.equal(other, first)


def test_empty_calls(pkg, dev):
    c = make_case([3], [20], 2, 2, 64, BF)
    got = call(pkg, dev, c, q=c.q[:0], tree_mask=c.mask[:0],
               cu_seqlens_q=torch.zeros(2, dtype=torch.int32))
    assert got.shape == (0, 2, 64)
    assert FP8  # (the fp8 cases are among SHAPES)


@pytest.mark.parametrize("hq,hkv,dim,nodes", [(2, 2, 128, [16, 7]), (4, 1, 64, [40, 12]),
                                              (8, 2, 96, [9, 16])])
@pytest.mark.parametrize("low,high", [(-26, -22), (-20, 4), (2, 6)])
def test_value_scales_of_any_size(pkg, dev, hq, hkv, dim, nodes, low, high):
    """fp16 rows over per-vector scales far from 1, and over scales that differ widely."""
    c = make_case(nodes, [515, 96], hq, hkv, dim, HF, "fp8_vector", seed=50 + dim)
    g = torch.Generator().manual_seed(dim)
    exps = low + (high - low) * torch.rand(c.v_scale.shape, generator=g)
    c.v_scale = torch.where(c.v_scale.isnan(), c.v_scale, torch.exp2(exps))
    check(call(pkg, dev, c), c, fine=True)


def flat_keys(c, weight):
    """Keys and values of sequence 0: position 0 has score 0 and value 0, each other one the
    weight ``weight`` next to it and value 1."""
    c.q.fill_(0)
    c.q[..., 0] = 8
    c.k.fill_(0)
    c.k[..., 0] = math.log(weight) * math.sqrt(c.q.shape[-1]) / 8
    c.v.fill_(1)
    blk = int(c.tables[0, 0])
    c.k[blk, 0], c.v[blk, 0] = 0, 0


@pytest.mark.parametrize("nodes", [[3], [40]])
def test_many_small_weights(pkg, dev, nodes):
    """fp16: 20000 keys of weight 1.4 2^-25 next to one of 1 are a part of the row."""
    c = make_case(nodes, [20000], 2, 1, 64, HF, seed=3, bits=[[1 << i for i in range(nodes[0])]])
    flat_keys(c, 1.4 * 2.0 ** -25)
    check(call(pkg, dev, c), c, fine=True)


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (HF, 64), (BF, 80)])
@pytest.mark.parametrize("scale", [0.0, -1 / 60.0])
def test_key_scale_zero_or_negative(pkg, dev, dtype, dim, scale):
    c = make_case([16, 40], [515, 96], 4, 2, dim, dtype, "fp8", seed=60)
    c.k_scale = torch.tensor(scale)
    check(call(pkg, dev, c), c)


def test_no_table_at_all(pkg, dev):
    """Tables of width 0 hold no position: rows of zeros."""
    c = make_case([3, 2], [40, 20], 4, 2, 128, BF)
    got = call(pkg, dev, c, block_tables=c.tables[:, :0])
    assert got.shape == c.q.shape and (got == 0).all()


def test_calls_side_by_side(pkg, dev):
    """Two streams, each with calls of its own: every call has its own partials."""
    cases = [make_case([26, 9], [2600, 511], 16, 4, 128, BF, seed=30),
             make_case([16, 7], [1515, 3096], 16, 8, 128, BF, "fp8", seed=31)]
    want = [call(pkg, dev, c) for c in cases]
    kernel = pkg.create_backend("auto", dev, BF, 128, 16)
    args = []
    for c in cases:
        args.append([x.to(dev) if x is not None else None
                     for x in (c.q, c.k, c.v, c.tables, c.lengths, c.cu, c.mask, c.k_scale, c.v_scale)])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                a = args[i]
                got[i].append(kernel.tree(*a[:6], cases[i].max_q, *a[6:]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
