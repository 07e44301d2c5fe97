"""Acceptance along draft trees on the GPU, sampled and greedy, against the plain rounds."""

import math

import pytest
import torch

from tests.tree_cases import ancestor_bits, pack_bits
from tests.tree_rounds import greedy_tree, random_trees, sampled_inputs, tree_accept

pytestmark = pytest.mark.gpu


def to(dev, args):
    return [x.to(dev) for x in args]


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b), (a.cpu(), b)


@pytest.mark.parametrize("n,w,vocab", [
    (1, 0, 1), (3, 0, 50), (1, 1, 2), (5, 3, 7), (8, 8, 1000), (4, 15, 16383), (4, 9, 16384),
    (3, 9, 16385), (6, 31, 5001), (2, 7, 49152), (3, 4, 65537), (2, 3, 152064), (2, 255, 300),
    (300, 4, 33)])
def test_sampled_rounds(pkg, dev, n, w, vocab):
    args = sampled_inputs(n, w, vocab, seed=n + w + vocab)
    got = pkg.tree_accept(*to(dev, args))
    want = tree_accept(*args)
    same(got, want)
    if n * w >= 30:
        assert want[2].max() >= 1 and not want[4].any()


@pytest.mark.parametrize("sharp,noise", [(0.0, 0.0), (1.0, 6.0), (12.0, 1.0), (30.0, 30.0)])
def test_sampled_rounds_of_other_distributions(pkg, dev, sharp, noise):
    """q = p (every first child accepted), far apart, and peaked with underflowed tails."""
    args = sampled_inputs(12, 12, 3001, seed=4, sharp=sharp, noise=noise)
    same(pkg.tree_accept(*to(dev, args)), tree_accept(*args))


@pytest.mark.parametrize("vocab", [8191, 8193, 32768, 32770, 40961, 49152, 49155, 100003])
def test_many_rejections_at_one_node(pkg, dev, vocab):
    """Passes over rows that are kept on the chip from the first one, wholly and in part; the
    same after an accepted draft."""
    args = list(sampled_inputs(4, 9, vocab, seed=vocab, noise=2.0))
    args[1][:] = torch.tensor([0, 0, 0, 0, 0, 5, 5, 5, 5])
    args[5][:] = 1 - 2.0 ** -20
    args[5][2:, 4] = 0  # the fifth draft is accepted, if anything is left for it
    args[2][:] = torch.tensor([9, 3, 9, 7])
    for r in range(4):
        for j in range(9):
            node = int(args[1][r, j])
            args[0][r, j] = int((args[3][r, node] - args[4][r, node] * (j != 4) * 3).argmax()) if j != 4 \
                else int((args[4][r, node] - 9 * args[3][r, node]).argmax())
    want = tree_accept(*args)
    same(pkg.tree_accept(*to(dev, args)), want)
    assert want[2][1] == 0 and want[2].max() == 1 and not want[4].any()


def test_uniforms_at_their_ends(pkg, dev):
    args = list(sampled_inputs(6, 9, 500, seed=5))
    top = 1 - 2.0 ** -24
    for a, f in ((0.0, 0.0), (top, top), (top, 0.0), (0.0, top)):
        args[5] = torch.full_like(args[5], a)
        args[6] = torch.full_like(args[6], f)
        same(pkg.tree_accept(*to(dev, args)), tree_accept(*args))


def test_zero_weights_are_never_drawn(pkg, dev):
    """Rows with long runs of zeros, also at both ends."""
    args = list(sampled_inputs(8, 6, 40000, seed=6))
    for x in (args[3], args[4]):
        x[..., :17000] = 0
        x[..., 17400:] = 0
        x[..., 17100:17200] = 0
        x /= x.sum(-1, keepdim=True)
    args[0] = 17000 + args[0] % 100
    got = pkg.tree_accept(*to(dev, args))
    same(got, tree_accept(*args))
    drawn = args[4][torch.arange(8), got.path.cpu().gather(1, got.accepted.cpu()[:, None])[:, 0],
                    got.final.cpu()]
    assert (drawn > 0).all()


def test_repeated_siblings_and_unreachable_drafts(pkg, dev):
    """The same token twice under one node; parents that are no earlier node."""
    args = list(sampled_inputs(40, 6, 12, seed=7, noise=2.0))
    args[1][:] = torch.tensor([0, 0, 0, 9, -1, 4])
    args[0][:, 1] = args[0][:, 0]
    args[2][:] = 6
    same(pkg.tree_accept(*to(dev, args)), tree_accept(*args))
    logits = args[4].log()
    want = greedy_tree(args[0], args[1], args[2], logits)
    same(pkg.greedy_tree_accept(*to(dev, args[:3]), logits.to(dev)), want)


def test_errors_are_flagged(pkg, dev):
    args = list(sampled_inputs(9, 3, 100, seed=8))
    tokens, parents, drafts, q, p, ua, uf = args
    parents[:] = torch.tensor([0, 0, 0])
    drafts[:] = 3
    ua[:] = 1 - 2.0 ** -24
    drafts[0] = 4                       # more drafts than columns
    drafts[1] = -1
    tokens[2, 0] = 100                  # outside the vocabulary
    tokens[3, 0] = -1
    q[4, 0, tokens[4, 0]] = 0           # cannot have been proposed
    p[5, 0, tokens[5, 0]] = math.nan
    p[6, 0, (tokens[6, 0] + 1) % 100] = math.nan   # spoils what a rejection leaves
    ua[6, 0] = 0.999
    q[6, 0, tokens[6, 0]] = 0.9
    p[7, 0] = 0                         # nothing to draw from
    drafts[8] = 0
    p[8, 0, 5] = math.inf
    want = tree_accept(*args)
    same(pkg.tree_accept(*to(dev, args)), want)
    assert want[4].all() and (want[3] == 0).all()


def test_rows_that_the_walk_does_not_visit_have_no_effect(pkg, dev):
    args = list(sampled_inputs(5, 10, 400, seed=9))
    want = tree_accept(*args)
    for r in range(5):
        visited = set(want[0][r].tolist())
        for i in range(11):
            if i not in visited:
                args[4][r, i] = math.nan
                if i < 10:
                    args[3][r, i] = math.nan
    same(pkg.tree_accept(*to(dev, args)), want)


def test_a_chain_is_the_chain_round(pkg, dev):
    args = list(sampled_inputs(16, 5, 2000, seed=10))
    args[1][:] = torch.arange(5)
    g = torch.Generator().manual_seed(1)
    for j in range(5):
        args[0][:, j] = torch.multinomial(args[3][:, j], 1, generator=g)[:, 0]
    got = pkg.tree_accept(*to(dev, args))
    tokens, _, drafts, q, p, ua, uf = to(dev, args)
    chain = pkg.speculative_accept(tokens, drafts, q, p, ua, uf)
    assert torch.equal(got.tokens, chain.tokens) and torch.equal(got.accepted, chain.accepted)
    assert torch.equal(got.final, chain.final) and not got.error.any()


def test_emitted_tokens_follow_the_target(pkg, dev):
    """First tokens of 200000 requests whose root has three drafts: within 5 standard
    deviations of p in every token (fixed seed)."""
    n, vocab = 200000, 6
    g = torch.Generator().manual_seed(11)
    q1 = torch.tensor([0.4, 0.3, 0.1, 0.1, 0.05, 0.05])
    p1 = torch.tensor([0.1, 0.35, 0.02, 0.23, 0.3, 0.0])
    q = q1.expand(n, 3, vocab).contiguous()
    p = p1.expand(n, 4, vocab).contiguous()
    tokens = torch.multinomial(q1.expand(n, vocab), 3, replacement=True, generator=g)
    parents = torch.zeros(n, 3, dtype=torch.int64)
    res = pkg.tree_accept(*to(dev, (tokens, parents, torch.full((n,), 3), q, p,
                                    torch.rand(n, 3, generator=g), torch.rand(n, generator=g))))
    share = torch.bincount(res.tokens[:, 0].cpu(), minlength=vocab).double() / n
    bound = 5 * (p1.double() * (1 - p1.double()) / n).sqrt()
    assert ((share - p1.double()).abs() <= bound).all() and not res.error.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,w,vocab", [(1, 0, 1), (3, 7, 9), (2, 16, 8191), (2, 5, 8192),
                                       (1, 6, 8193), (5, 31, 1000), (2, 255, 77),
                                       (1, 3, 151936)])
def test_greedy_rounds(pkg, dev, n, w, vocab, dtype):
    g = torch.Generator().manual_seed(n + w + vocab)
    # few distinct values: ties are common
    logits = (torch.randn(n, w + 1, vocab, generator=g) * 4).round().to(dtype)
    parents = random_trees(n, w, g)
    targets = greedy_tree(torch.zeros(n, w, dtype=torch.int64), parents, torch.zeros(n), logits)[0]
    tokens = targets.gather(1, parents) if w else torch.zeros(n, 0, dtype=torch.int64)
    other = torch.randint(0, vocab, (n, w), generator=g)
    tokens = torch.where(torch.rand(n, w, generator=g) < 0.6, tokens, other)
    drafts = torch.randint(0, w + 1, (n,), generator=g)
    drafts[0] = w
    want = greedy_tree(tokens, parents, drafts, logits)
    same(pkg.greedy_tree_accept(*to(dev, (tokens, parents, drafts, logits))), want)


def test_greedy_extremes(pkg, dev):
    """NaN first, signed zeros equal, rows of one value, of -inf and of the lowest number."""
    logits = torch.zeros(1, 6, 300)
    logits[0, 0, 7] = -0.0
    logits[0, 1, 40] = math.nan
    logits[0, 1, 3] = math.inf
    logits[0, 1, 90] = math.nan
    logits[0, 2] = -math.inf
    logits[0, 3] = torch.finfo(torch.float32).min
    logits[0, 4] = -1.0
    logits[0, 4, 299] = -0.5
    logits[0, 5] = torch.arange(300.0)
    tokens = torch.tensor([[0, 40, 0, 0, 299]])
    parents = torch.arange(5)[None]
    drafts = torch.tensor([5])
    targets, path, accepted, last = pkg.greedy_tree_accept(*to(dev, (tokens, parents, drafts, logits)))
    assert targets.tolist() == [[0, 40, 0, 0, 299, 299]]
    assert accepted.tolist() == [5] and last.tolist() == [299]
    # a chain is the chain's greedy round
    chain = pkg.greedy_accept_batched(tokens.to(dev), drafts.to(dev), logits.to(dev))
    assert torch.equal(chain[0], targets) and torch.equal(chain[1], accepted)


def test_greedy_strided_and_unaligned_rows(pkg, dev):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 5, 1100, generator=g).bfloat16().to(dev)
    logits = wide[:, :, 3:1004]
    parents = random_trees(2, 4, g)
    tokens = torch.randint(0, 1001, (2, 4), generator=g)
    drafts = torch.tensor([4, 9])  # a count past the columns is cut
    got = pkg.greedy_tree_accept(*to(dev, (tokens, parents, drafts)), logits)
    same(got, greedy_tree(tokens, parents, drafts, logits.cpu()))


def test_rounds_in_a_graph(pkg, dev):
    args = to(dev, sampled_inputs(7, 12, 3000, seed=12))
    logits = args[4].log()
    eager = pkg.tree_accept(*args)
    greedy = pkg.greedy_tree_accept(*args[:3], logits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = pkg.tree_accept(*args)
        b = pkg.greedy_tree_accept(*args[:3], logits)
    for _ in range(3):
        for x in (*a, *b):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*a, *b), (*eager, *greedy)))
        assert math.isfinite(torch.randn(1 << 18, device=dev).sum().item())
    # new uniforms in place
    args[5].copy_(torch.rand(7, 12, device=dev))
    graph.replay()
    torch.cuda.synchronize()
    again = pkg.tree_accept(*args)
    assert all(torch.equal(x, y) for x, y in zip(a, again))


def test_tree_masks(pkg, dev):
    g = torch.Generator().manual_seed(2)
    counts = [1, 5, 0, 140, 3]
    w = 200
    parents = torch.full((5, w), 77, dtype=torch.int64)
    rows = []
    for s, m in enumerate(counts):
        if m:
            up = random_trees(1, m - 1, g)[0]
            parents[s, :m - 1] = up
            rows += ancestor_bits(up.tolist())
    cu = torch.tensor([0, 1, 6, 6, 146, 149], dtype=torch.int32)
    got = pkg.tree_masks(parents.to(dev), cu.to(dev), 152)
    assert got.shape == (152, 4)
    assert torch.equal(got[:149].cpu(), pack_bits(rows, 4)) and (got[149:] == 0).all()
    # a parent that is no earlier node ends the walk
    bad = torch.tensor([[0, 5, 2, -3]])
    got = pkg.tree_masks(bad.to(dev), torch.tensor([0, 5], dtype=torch.int32).to(dev), 5)
    assert got[:, 0].tolist() == [1, 3, 4, 12, 16]
    assert pkg.tree_masks(bad[:0].to(dev), cu[:1].to(dev), 3).eq(0).all()


def test_tree_masks_of_single_nodes(pkg, dev):
    """No drafts at all; sequences of one node; rows before the first sequence and behind the last."""
    cu = torch.tensor([2, 3, 4, 4, 5], dtype=torch.int32)
    got = pkg.tree_masks(torch.zeros(4, 0, dtype=torch.int64, device=dev), cu.to(dev), 9)
    assert got.tolist() == [[0], [0], [1], [1], [1], [0], [0], [0], [0]]
    got = pkg.tree_masks(torch.zeros(4, 70, dtype=torch.int64, device=dev), cu.to(dev), 3)
    assert got.tolist() == [[0, 0], [0, 0], [1, 0]]


def test_rounds_on_two_streams(pkg, dev):
    """Calls in flight side by side."""
    args = [to(dev, sampled_inputs(20, 9, 30000, seed=s)) for s in (1, 2)]
    logits = [a[4].log() for a in args]
    want = [(pkg.tree_accept(*a), pkg.greedy_tree_accept(*a[:3], x)) for a, x in zip(args, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((pkg.tree_accept(*args[i]), pkg.greedy_tree_accept(*args[i][:3], logits[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            for x, y in zip(pair, want[i]):
                assert all(torch.equal(a, b) for a, b in zip(x, y))
