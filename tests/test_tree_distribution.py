"""The distribution of the first token behind a root whose children are verified (the oracle's rules), exactly: summed over
all drafts with their probabilities and integrated over the uniform numbers, whose thresholds are found by bisection."""
import itertools

import pytest
import torch

from oracle import tree_oracle as O

EPS = 2.0 ** -48


def threshold(holds):
    """The u in [0, 1] up to which holds(u), which does not come back once it is lost."""
    if not holds(0.0):
        return 0.0
    lo, hi = 0.0, 1.0
    if holds(1.0 - EPS):
        return 1.0
    while hi - lo > EPS:
        mid = (lo + hi) / 2
        lo, hi = (mid, hi) if holds(mid) else (lo, mid)
    return lo


def first_token(p, q, n):
    """P(token) of n children; drawn from q, or (q None) the tokens 1, 0, 1, ... taken as given."""
    V = len(p)
    rows = torch.tensor([p] * (n + 1), dtype=torch.float64)
    draft = None if q is None else torch.tensor([q] * (n + 1), dtype=torch.float64)
    tree, out = [-1] + [0] * n, [0.0] * V
    drafts = [tuple((j + 1) % 2 for j in range(n))] if q is None else itertools.product(range(V), repeat=n)
    for x in drafts:
        weight = 1.0
        for t in x:
            weight *= 1.0 if q is None else q[t]
        if weight == 0:
            continue

        def run(u, u_next=0.0):
            return O.verify(tree, [0, *x], rows, [0.0, *u, *[1.0] * (n - len(u))], u_next, draft)

        u = []  # numbers at which the children so far are rejected
        for j in range(n):
            t = threshold(lambda z: run(u + [z])[0] == [0, j + 1])
            out[x[j]] += weight * t
            weight *= 1 - t
            if t == 1.0:
                break
            u.append(1.0)
        else:
            at = 0.0
            for token in range(V):  # the tokens rise with u_next
                t = threshold(lambda z: run(u, z)[1] <= token)
                out[token] += weight * max(t - at, 0.0)
                at = max(at, t)
    return out


@pytest.mark.parametrize("n", [1, 2, 3])
@pytest.mark.parametrize("q", [None, [0.2, 0.5, 0.3], [0.0, 0.9, 0.1], [0.5, 0.2, 0.3]])
@pytest.mark.parametrize("p", [[0.5, 0.2, 0.3], [0.25, 0.75, 0.0], [0.0, 0.0, 1.0]])  # (the last two as filtered and normalised again)
def test_tokens_have_the_targets_distribution(p, q, n):
    got = first_token(p, q, n)
    assert all(abs(a - b) < 1e-9 for a, b in zip(got, p)), got


def test_rows_that_do_not_sum_to_one():
    """The rules take a row as it is: with a sum of 1/2 a given token is accepted half as often as it weighs. Rows are to sum to 1."""
    got = first_token([0.25, 0.25, 0.0], None, 1)
    assert got == pytest.approx([0.75, 0.25, 0.0], abs=1e-9)
