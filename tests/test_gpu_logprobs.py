"""Token log probabilities on the GPU against float64 log softmax."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(x, tokens, top_n):
    """(logprob, rank, entropy, top_logprob, top_tokens) and tolerances of the first three
    kinds of numbers, in float64.

    With d = x - m taken in float32 (off by 2^-24 |d|), the exponent d log2(e) in float32 (its
    constant and its product off by 1.3 2^-24 of it) and an exponential of two half steps, a
    weight e^d is off by (2 + 2.3 |d|) 2^-24 of itself; two float32 additions of weights add two
    half steps before the float64 sums S and T.  log S is then off by E (4 + 2.3 |d|) 2^-24 with E
    the mean under the row's distribution, T / S (one more product) by E |d| (5 + 2.3 |d|) + E |d|
    E (4 + 2.3 |d|), and an output is rounded once.
    """
    x = x.double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    d = (x - x.amax(-1, keepdim=True)).abs()
    w = torch.where(p > 0, d, torch.zeros_like(d))
    mean = lambda f: (p * f).sum(-1)  # noqa: E731
    u = 2.0 ** -24
    e_lse = u * mean(4 + 2.3 * w) * 1.1
    e_t = u * (mean(w * (5 + 2.3 * w)) + mean(w) * mean(4 + 2.3 * w)) * 1.1
    at = torch.arange(x.shape[0])
    order = x.sort(dim=-1, descending=True, stable=True).indices
    rank = (order == tokens[:, None]).nonzero()[:, 1] + 1
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    top = order[:, :top_n]
    tl = lp.gather(1, top)
    got = lp[at, tokens]
    return (got, rank, entropy, tl, top), (e_lse + u * got.abs(), e_lse + e_t + u * entropy.abs(),
                                           e_lse[:, None] + u * tl.abs())


def check(res, x, tokens, top_n):
    (lp, rank, ent, tl, top), (a, b, c) = plain(x.float().cpu(), tokens.cpu(), top_n)
    assert torch.equal(res.rank.cpu(), rank)
    assert torch.equal(res.top_tokens.cpu(), top)
    for got, want, tol in ((res.logprob, lp, a), (res.entropy, ent, b), (res.top_logprob, tl, c)):
        got = got.double().cpu()
        same = got == want  # (infinities)
        assert (same | ((got - want).abs() <= tol)).all(), float((got - want).abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,vocab,top_n", [
    (1, 1, 1), (1, 1, 0), (3, 5, 5), (7, 64, 64), (2, 2047, 20), (2, 2048, 1), (2, 2049, 64),
    (40, 8191, 20), (40, 8192, 5), (40, 8193, 64), (5, 49152, 20), (60, 49152, 3),
    (1, 151936, 64), (17, 152064, 20), (300, 1000, 10)])
def test_matches_plain(pkg, dev, m, vocab, top_n, dtype):
    g = torch.Generator().manual_seed(m + vocab + top_n)
    x = (torch.randn(m, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (m,), generator=g)
    tokens[0] = int(x[0].float().argmax())
    check(pkg.token_logprobs(x.to(dev), tokens.to(dev), top_n=top_n), x, tokens, top_n)


@pytest.mark.parametrize("vocab", [600, 30000, 300000, 1 << 20])
def test_ties_and_orders(pkg, dev, vocab):
    """Equal logits by ascending column: constant rows, two values, rising, falling, blocks."""
    c = torch.arange(vocab, dtype=torch.float32)
    rows = [torch.zeros(vocab), (c % 2), c / vocab, -c / vocab, (c % 97 == 3).float(),
            torch.where(c % 3 == 0, 0.0, -0.0), (c // 32 % 7 == 2).float() * 5]
    x = torch.stack(rows)
    tokens = torch.tensor([vocab - 1, 4, vocab - 1, 0, 3, vocab // 2, vocab - 5])
    check(pkg.token_logprobs(x.to(dev), tokens.to(dev), top_n=30), x, tokens, 30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top_n", [1, 5, 20, 64])
def test_uneven_rows(pkg, dev, dtype, top_n):
    """The largest columns side by side, at the row's start, its end and within a wave's columns;
    a row's end inside the first wave's columns; fewer columns above -inf than asked for."""
    g = torch.Generator().manual_seed(top_n)
    for vocab in (2048 * 5 + 384, 8192 * 3 + 100, 70):
        x = torch.randn(6, vocab, generator=g)
        x[0, :min(200, vocab)] += 20
        x[1, -40:] += 20
        x[2, vocab // 2:vocab // 2 + 30] += 20
        x[3, :] = -math.inf
        x[3, 3::vocab // 7] = 1.0
        x[4, :vocab - 300 if vocab > 300 else 1] = -50.0
        x = x.to(dtype)
        tokens = torch.tensor([0, vocab - 1, vocab // 2, 3, 0, 1])
        check(pkg.token_logprobs(x.to(dev), tokens.to(dev), top_n=top_n), x, tokens, top_n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_logits(pkg, dev, dtype):
    """-inf and the type's lowest value as masks; a dominant token; one token left."""
    g = torch.Generator().manual_seed(0)
    low = torch.finfo(dtype).min
    x = (torch.randn(6, 20000, generator=g) * 3).to(dtype)
    x[0, 100:] = -math.inf
    x[1, :19000] = -math.inf
    x[2, 5:] = low
    x[3] = -math.inf
    x[3, 17] = -30.0
    x[4, 9] = 60.0
    x[5] = low
    tokens = torch.tensor([3, 19500, 2, 17, 9, 44])
    check(pkg.token_logprobs(x.to(dev), tokens.to(dev), top_n=20), x, tokens, 20)
    # a masked token's own probability is 0
    res = pkg.token_logprobs(x[:1].to(dev), torch.tensor([500], device=dev), top_n=2)
    assert res.logprob.item() == -math.inf and res.rank.item() == 501


def test_rows_that_are_no_distribution(pkg, dev):
    x = torch.randn(4, 9000)
    x[0, 8500] = math.nan
    x[1, 33] = math.inf
    x[2] = -math.inf
    tokens = torch.tensor([8500, 33, 7, 8])
    res = pkg.token_logprobs(x.to(dev), tokens.to(dev), top_n=3)
    assert torch.isnan(res.logprob[:3]).all() and torch.isnan(res.entropy[:3]).all()
    assert torch.isnan(res.top_logprob[:3]).all() and torch.isfinite(res.top_logprob[3]).all()
    # the order still holds: NaN first, equal logits by column
    assert res.rank.tolist()[:3] == [1, 1, 8]
    assert res.top_tokens[0, 0].item() == 8500 and res.top_tokens[1, 0].item() == 33
    assert res.top_tokens[2].tolist() == [0, 1, 2]


def test_row_indices_and_tokens_out_of_range(pkg, dev):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 700, generator=g).to(dev)
    rows = torch.tensor([3, -1, 3, 6, 0, 5, 1 << 40], device=dev)
    tokens = torch.tensor([8, 1, 700, 2, -1, 699, 0], device=dev)
    res = pkg.token_logprobs(x, tokens, rows=rows, top_n=4)
    ok = [0, 5]
    (lp, rank, _, _, _), (tol, _, _) = plain(x[rows[ok]].cpu(), tokens[ok].cpu(), 4)
    assert ((res.logprob[ok].double().cpu() - lp).abs() <= tol).all()
    assert res.rank[ok].cpu().equal(rank)
    none = [1, 3, 6]
    assert torch.isnan(res.logprob[none]).all() and torch.isnan(res.entropy[none]).all()
    assert (res.rank[none] == 0).all() and (res.top_tokens[none] == -1).all()
    assert torch.isnan(res.top_logprob[none]).all()
    token = [2, 4]  # the row holds, the token does not
    assert torch.isnan(res.logprob[token]).all() and (res.rank[token] == 0).all()
    assert torch.isfinite(res.entropy[token]).all()
    assert res.top_tokens[2].equal(res.top_tokens[0])
    assert res.entropy[2] == res.entropy[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_rows(pkg, dev, dtype):
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(9, 5003, generator=g).to(dtype).to(dev)
    x = wide[::2, 1:4000]
    tokens = torch.randint(0, 3999, (5,), generator=g).to(dev)
    check(pkg.token_logprobs(x, tokens, top_n=9), x, tokens, 9)


def test_many_rows_and_none(pkg, dev):
    g = torch.Generator().manual_seed(7)
    x = torch.randn(70000, 5, generator=g)
    tokens = torch.randint(0, 5, (70000,), generator=g)
    check(pkg.token_logprobs(x.to(dev), tokens.to(dev), top_n=2), x, tokens, 2)
    rows = torch.randint(0, 70000, (66000,), generator=g)
    check(pkg.token_logprobs(x.to(dev), tokens[:66000].to(dev), rows=rows.to(dev), top_n=1),
          x[rows], tokens[:66000], 1)
    res = pkg.token_logprobs(x[:0].to(dev), tokens[:0].to(dev), top_n=2)
    assert res.logprob.shape == (0,) and res.top_tokens.shape == (0, 2)


def test_offsets_past_32_bits(pkg, dev):
    """Rows behind the first 2^32 elements."""
    m = (1 << 32) // 100000 + 3
    big = torch.empty(m, 100000, dtype=torch.bfloat16, device=dev)
    big[-2:] = torch.randn(2, 100000, device=dev).bfloat16()
    tokens = torch.tensor([99999, 5], device=dev)
    res = pkg.token_logprobs(big, tokens, rows=torch.tensor([m - 1, m - 2], device=dev), top_n=3)
    check(res, big[[m - 1, m - 2]].float(), tokens, 3)


def test_in_a_graph_and_bit_for_bit(pkg, dev):
    g = torch.Generator().manual_seed(8)
    x = torch.randn(5, 50000, generator=g).bfloat16().to(dev)
    tokens = torch.randint(0, 50000, (5,), generator=g).to(dev)
    eager = pkg.token_logprobs(x, tokens, top_n=20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.token_logprobs(x, tokens, top_n=20)
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        assert math.isfinite(torch.randn(1 << 18, device=dev).sum().item())


def test_one_row_for_many_tokens(pkg, dev):
    """The same row index, and the same token, several times; on a stream of its own."""
    g = torch.Generator().manual_seed(30)
    x = torch.randn(3, 20000, generator=g) * 3
    rows = torch.tensor([2, 2, 0, 2, 0])
    tokens = torch.tensor([5, 5, 5, 19999, 7])
    xd, rd, td = x.to(dev), rows.to(dev), tokens.to(dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        res = pkg.token_logprobs(xd, td, rows=rd, top_n=8)
    torch.cuda.synchronize()
    check(res, x[rows], tokens, 8)
    assert res.logprob[0] == res.logprob[1]
