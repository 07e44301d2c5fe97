"""The final draw of a sampled tree round where next to nothing is left of the target."""

from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu


def row_with_rest(pa, qa, mass, vocab, at):
    """A row of p and q, of dyadic numbers, whose weights after one rejection, max(p - q, 0), sum to
    ``mass - 1`` exactly: column ``at`` holds (pa, qa), four others what is missing, so that nothing
    of theirs is left after the second rejection.  Column 0 has draft mass only."""
    p, q = torch.zeros(vocab), torch.zeros(vocab)
    q[0] = 0.25
    p[at], q[at] = float(pa), float(qa)
    first = torch.tensor(float(pa)) - torch.tensor(float(qa))  # rounded to float32
    rest = (mass - 1 - Fraction(float(first))) * 2 ** 52
    assert rest.denominator == 1 and 0 < rest < 2 ** 52
    for i in range(4):
        digits = (int(rest) >> (13 * i)) & 0x1FFF
        col = at + 4 * (i + 1)
        q[col] = 4 * 2.0 ** (13 * (i + 1) - 52)
        p[col] = float(q[col]) + digits * 2.0 ** (13 * i - 52)
        assert float(p[col]) - float(q[col]) == digits * 2.0 ** (13 * i - 52)
    return p, q


@pytest.mark.parametrize("pa,qa", [("1507393/2097152", "8049737/16777216"),
                                   ("11507597/16777216", "13361213/33554432"),
                                   ("2604201/4194304", "6985153/16777216"),
                                   ("5918039/8388608", "15537223/33554432")])
@pytest.mark.parametrize("vocab,at", [(64, 5), (70001, 69001)])
def test_no_token_without_weight(pkg, dev, pa, qa, vocab, at):
    """Two drafts of column 0, which p does not hold, are rejected; C = 1 + R is then p / q of one
    column rounded up to 2^-52, and every other column's rest is below 0.  Whether that column's
    counts as 2^-50 or as nothing, no other token may come out."""
    pa, qa = Fraction(pa), Fraction(qa)
    mass = Fraction(-((-pa * 2 ** 52) // qa), 2 ** 52)
    p0, q0 = row_with_rest(pa, qa, mass, vocab, at)
    p = torch.stack([p0, torch.full((vocab,), 1 / vocab), torch.full((vocab,), 1 / vocab)])[None]
    q = torch.stack([q0, torch.full((vocab,), 1 / vocab)])[None]
    zeros = torch.zeros(1, 2, dtype=torch.int64)
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        args = (zeros, zeros, torch.tensor([2]), q, p, torch.full((1, 2), 0.5), torch.tensor([u]))
        res = pkg.tree_accept(*(x.to(dev) for x in args))
        assert int(res.accepted) == 0
        assert bool(res.error) or int(res.final) == at
        assert int(res.tokens[0, 0]) == int(res.final)
