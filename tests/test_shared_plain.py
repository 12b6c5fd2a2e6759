"""The float64 forms that the kernels of shared and chosen pages are compared with, on numbers worked out by hand."""
import math

import torch

import plain_pages as P
from plain_pages import F, PAGE, Paged

LN2 = math.log(2.0)


def rows(*lens, heads=2):
    """Rows of one new token each behind these contexts, features of two, keys of zero and values of zero wherever a token is."""
    case = Paged([(n, 1) for n in lens], heads, 1, 2, seed=1)
    case.k[~case.k.isnan()] = 0.0
    case.v[~case.v.isnan()] = 0.0
    case.q[:] = 0.0
    return case


def close(got, want):
    return torch.allclose(got, torch.tensor(want, dtype=F), rtol=1e-14, atol=0.0)


def test_weights_are_powers_of_the_scores():
    """Scores 0, 1, 2 at a scale of ln 2 weigh 1, 2, 4: (7 + 2 * 7 + 4 * 14) / 7 = 11; the second head's query is turned round: (4 * 7 + 2 * 7 + 14) / 7 = 8."""
    case = rows(2)
    page = int(case.table[0, 0])
    case.k[page, 0, :3, 0] = torch.tensor([0.0, 1.0, 2.0])
    case.v[page, 0, :3, 0] = torch.tensor([7.0, 7.0, 14.0])
    case.v[page, 0, :3, 1] = torch.tensor([7.0, -7.0, 0.0])
    case.q[0] = torch.tensor([1.0, 0.0, -1.0, 0.0])
    out, size = P.shared(case, LN2)
    assert close(out, [[11.0, -1.0, 8.0, 2.0]]) and close(size, [[11.0, 3.0, 8.0, 6.0]])


def test_pages_that_are_not_there_and_positions_before_everything():
    """Equal weights: a mean over what is there.  Values 1 on the row's first page, 2 on the second, 3 at its last two places."""
    case = rows(129)
    for p, v in enumerate((1.0, 2.0, 3.0)):
        page = case.v[int(case.table[0, p])]
        page[~page.isnan()] = v
    assert close(P.shared(case, 1.0)[0], [[(64 + 2 * 64 + 3 * 2) / 130] * 4])
    case.table[0, 1] = -1
    assert close(P.shared(case, 1.0)[0], [[(64 + 3 * 2) / 66] * 4])
    case.table[0] = -1
    assert close(P.shared(case, 1.0)[0], [[0.0] * 4])
    case = rows(129)
    case.tok_pos[0] = -1
    assert close(P.shared(case, 1.0)[0], [[0.0] * 4])


def test_lists():
    """The same row: pages as often as they are listed, up to the token's position, and as many entries as pages up to it."""
    case = rows(129)
    for p, v in enumerate((1.0, 2.0, 3.0)):
        page = case.v[int(case.table[0, p])]
        page[~page.isnan()] = v
    for entries, mean in (([2, 0, -1], (64 + 6) / 66), ([0, 0, 1], (128 + 128) / 192), ([-1, -1, -1, 0], 0.0), ([7, 3, 2, 1], 3.0), ([1], 2.0)):
        assert close(P.listed(case, [[entries]], 1.0)[0], [[mean] * 4]), entries


def test_bounds():
    """a = 4: codes rint(x * 31.75): 0.5 -> 16, 1 -> 32, 4 -> 127, -2 -> -63.5 and so -64.  A page of zeros has the smallest a."""
    case = rows(1, 1)
    page = int(case.table[0, 0])
    case.k[page, 0, :2] = torch.tensor([[1.0, -2.0], [0.5, 4.0]])
    codes, scale = P.bounds(case, 0, 0, 2)
    assert codes.tolist() == [[[16.0, -64.0], [32.0, 127.0]]] and scale.tolist() == [float(torch.tensor(4.0 / 127.0))]
    codes, scale = P.bounds(case, 0, 0, 1)                  # (the first token alone, a = 2)
    assert codes.tolist() == [[[64.0, -127.0], [64.0, -127.0]]]
    codes, scale = P.bounds(case, 1, 0, 2)
    assert codes.tolist() == [[[0.0, 0.0], [0.0, 0.0]]] and float(scale) > 0.0


def test_choice():
    """q = (1, -1): codes 127 and -127, so that a page's score goes by its highest first feature less its lowest second one; the second head's query is zero."""
    case = rows(5 * PAGE)
    case.q[0] = torch.tensor([1.0, -1.0, 0.0, 0.0])
    codes = torch.zeros(case.k.shape[0], 1, 2, 2, dtype=torch.int8)
    scales = torch.ones(case.k.shape[0], 1)
    for p, (low, high) in enumerate(((0, 3), (-9, 0), (1, 5), (-4, 5), (-8, 1), (0, 0))):            # scores of 3, 9, 4, 9, 9, 0
        codes[int(case.table[0, p]), 0] = torch.tensor([[0, low], [high, 99]])
    pick = lambda *a: P.choose(case, codes, scales, 0, *a)[0]  # noqa: E731
    assert pick(3, 0, 1) == [1, 3, 5]                       # the last one, and of equal scores the lower pages
    assert pick(2, 1, 1) == [0, 5]
    assert pick(1, 1, 1) == [0]                             # fewer than must be: the lowest
    assert pick(4, 1, 2) == [0, 1, 4, 5]
    assert pick(8, 0, 1) == [0, 1, 2, 3, 4, 5, -1, -1]
    scales[int(case.table[0, 3])] = 2.0                     # a score of 18
    assert pick(2, 0, 1) == [3, 5]
    scales[int(case.table[0, 2])] = math.inf                # keys that are not finite come before scores
    assert pick(2, 0, 1) == [2, 5]
    case.table[0, 2] = -1                                   # pages that are not there are not taken
    assert pick(4, 0, 1) == [1, 3, 4, 5]
    case.tok_pos[0] = 2 * PAGE                              # of three pages two are there
    assert pick(3, 0, 1) == [0, 1, -1]
    case.tok_pos[0] = -1
    assert pick(2, 1, 1) == [-1, -1]
