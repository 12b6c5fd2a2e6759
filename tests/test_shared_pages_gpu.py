"""Attention over shared and over chosen pages, bounds of pages and the choice by them, on the GPU against float64.  How far results may be off is worked out in
``plain_pages.off`` from the roundings that the kernels make; bounds and chosen pages have to be equal."""
import math

import pytest
import torch

import plain_pages as P
from plain_pages import PAGE, Paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F = torch.float64


def K():
    from exl3_server_b200.ops import kernels
    return kernels


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def workspace():
    from exl3_server_b200.engine.batch import Workspace
    return Workspace(torch.device(DEV))


def wide(case, table):
    """The table with empty columns behind its own, so many that the call counts as one that reads more than 128 MB: those that read less leave groups alone."""
    pages = 128e6 / (len(case.rows) * -(-case.max_new * (case.h // case.g) // 16) * case.g * PAGE * case.d * 4)
    return torch.cat([table, torch.full((table.shape[0], int(pages) + 1), -1, dtype=torch.int32, device=table.device)], 1)


def run_shared(case, groups="own", ws=None, scale=None, q=None, little=False, **kw):
    groups = case.groups if groups == "own" else groups
    table = case.table.to(DEV)
    if groups and case.max_new and not little:
        table = wide(case, table)
    y = K().attn_shared(case.q.to(DEV) if q is None else q, case.k.to(DEV), case.v.to(DEV), table, ints(case.start), ints(case.pos0),
                        ints(groups).view(-1, 3) if groups is not None else None, case.max_new, case.h, case.g, case.d,
                        scale=case.d ** -0.5 if scale is None else scale, workspace=ws, **kw)
    torch.cuda.synchronize()
    K().check_status()
    return y


HEADS = [(16, 2, 64), (4, 4, 64), (8, 2, 128), (32, 2, 128), (7, 1, 128), (10, 2, 64), (32, 1, 128), (40, 1, 64)]


# ---- rows without groups: the walk alone --------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("rows", [[(0, 1)], [(63, 1), (64, 1), (0, 1)], [(700, 1), (5, 1), (1290, 1)], [(100, 3), (0, 2), (62, 5), (130, 1)], [(0, 0), (10, 1), (3, 0)]])
def test_walk(heads, kv_heads, d, rows):
    case = Paged(rows, heads, kv_heads, d, seed=len(rows) + d)
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, groups=None, ws=workspace()), want, size) <= 1.0


def test_walk_of_many_tokens():
    case = Paged([(70, 90), (0, 33), (500, 7)], 8, 2, 128, seed=3)
    want, size = P.shared(case, 0.07)
    assert P.off(run_shared(case, groups=None, scale=0.07), want, size) <= 1.0


# ---- groups ---------------------------------------------------------------------------------------------------------------------

def share(groups, loose=0):
    """[(rows, pages)] -> what Paged takes."""
    return [(j, p) for j, (n, p) in enumerate(groups) for _ in range(n)] + [None] * loose


@pytest.mark.parametrize("little", [False, True])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("groups,loose,own,new", [
    ([(1, 1)], 0, [0], [1]),                                # nothing but the new token behind one page
    ([(2, 3)], 0, [10, 77], [1, 1]),
    ([(3, 5), (2, 1)], 2, [0, 63, 64, 1, 200, 30, 0], [1, 1, 1, 1, 1, 1, 1]),
    ([(2, 9), (1, 4)], 1, [5, 0, 64, 40], [3, 1, 9, 2]),
])
def test_shared(heads, kv_heads, d, groups, loose, own, new, little):
    rows, shares = [], share(groups, loose)
    for s, c, n in zip(shares, own, new):
        rows.append(((s[1] * PAGE if s else 0) + c, n))
    case = Paged(rows, heads, kv_heads, d, share=shares, seed=d + len(rows))
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, ws=workspace(), little=little), want, size) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d,n,new", [(8, 2, 128, 70, 1), (4, 4, 64, 300, 1), (16, 1, 64, 20, 9), (6, 2, 128, 24, 13)])
def test_more_queries_than_a_tile(heads, kv_heads, d, n, new):
    case = Paged([(6 * PAGE + (i * 37) % 130, 1 + (i * 5) % new) for i in range(n)], heads, kv_heads, d, share=share([(n, 6)]), seed=1)
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 8, 64), (8, 8, 128)])
@pytest.mark.parametrize("pages", [[1], [1, 1, 2, 1, 3]])
def test_many_groups_of_few_pages(heads, kv_heads, d, pages):
    """A block has several tiles one behind the other, of which only one of its two sets of queries has a page."""
    shares = [(j, pages[j % len(pages)]) for j in range(60) for _ in range(16)]
    case = Paged([(p * PAGE + r % 7, 1) for r, (_, p) in enumerate(shares)], heads, kv_heads, d, share=shares, seed=8)
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 8, 64), (8, 8, 128)])
def test_many_groups_of_few_pages_beside_a_large_one(heads, kv_heads, d):
    """The same, where the two sets have places of their own for their queries."""
    shares = [(j, 1) for j in range(50) for _ in range(16)] + [(99, 2)] * 140
    case = Paged([(s[1] * PAGE + r % 7, 1) for r, s in enumerate(shares)], heads, kv_heads, d, share=shares, seed=9)
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


def test_long_prefix_and_many_blocks():
    case = Paged([(300 * PAGE + 5, 1), (300 * PAGE + 100, 2)], 8, 2, 64, share=share([(2, 300)]), seed=2)
    want, size = P.shared(case, 0.125)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (8, 2, 128), (6, 6, 128), (16, 1, 64), (5, 1, 128), (16, 2, 128)])
@pytest.mark.parametrize("rows,groups", [
    ([(0, 200)], []),                                       # a prompt
    ([(3, 130), (700, 65), (10, 1), (0, 300)], []),         # prompts beside a token, behind contexts
    ([(200, 150), (192, 70), (193, 2), (50, 129)], [(3, 3)]),                # behind shared pages, beside drafts
    ([(64, 17), (64, 16), (64, 33), (64, 1)], [(4, 1)]),
    ([(128, 400), (128, 3)], [(1, 2)]),
])
def test_rows_of_many_tokens(heads, kv_heads, d, rows, groups):
    case = Paged(rows, heads, kv_heads, d, share=share(groups, len(rows) - sum(n for n, _ in groups)), seed=d + len(rows))
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (8, 2, 128)])
def test_values_of_later_tokens_of_a_prompt(heads, kv_heads, d):
    """A prompt's tokens 70 and 100 have values that are not finite: those before them stay as they are, the others' features are not finite."""
    case = Paged([(40, 140), (20, 100)], heads, kv_heads, d, seed=26)
    want, size = P.shared(case, d ** -0.5)
    for at, feature, value in ((110, 3, math.nan), (140, 7, math.inf)):
        case.v[int(case.table[0, at // PAGE]), :, at % PAGE, feature] = value
    got = run_shared(case, ws=workspace()).cpu().view(-1, heads, d)
    w, s = want.view(-1, heads, d), size.view(-1, heads, d)
    for t in range(240):
        bad = {f for at, f in ((110, 3), (140, 7)) if t < 140 and 40 + t >= at}
        rest = [i for i in range(d) if i not in bad]
        assert P.off(got[t][:, rest], w[t][:, rest], s[t][:, rest]) <= 1.0, t
        assert all(not bool(torch.isfinite(got[t][:, f]).any()) for f in bad), t


# ---- bounds and the choice ----------------------------------------------------------------------------------------------------------

def make_bounds(case):
    """Bounds by the kernel, for all of the rows' tokens at once; pages that no row owns keep a pattern."""
    k = K()
    pages = case.k.shape[0]
    codes, scales = k.page_bounds_pool(pages, case.g, case.d, DEV)
    codes.fill_(99)
    scales.fill_(-5.0)
    lens = [c + n for c, n in case.rows]
    start = [sum(lens[:i]) for i in range(len(lens) + 1)]
    k.page_bounds(case.k.to(DEV), codes, scales, case.table.to(DEV), ints(start), ints([0] * len(lens)), max(lens + [0]))
    torch.cuda.synchronize()
    return codes, scales


@pytest.mark.parametrize("kv_heads,d", [(1, 64), (3, 64), (2, 128), (5, 128)])
@pytest.mark.parametrize("rows", [[(0, 1)], [(63, 1), (64, 1), (0, 130)], [(200, 5), (0, 0), (64, 64), (1000, 1)]])
def test_bounds(kv_heads, d, rows):
    case = Paged(rows, kv_heads, kv_heads, d, seed=d)
    codes, scales = make_bounds(case)
    low, high = K().page_bounds_load(codes, scales, ints(list(range(-1, codes.shape[0] + 1))))
    assert bool((low[[0, -1]] == 0).all() and (high[[0, -1]] == 0).all())
    seen = set()
    for r, (c, n) in enumerate(rows):
        for p in range(-(-(c + n) // PAGE)):
            page = int(case.table[r, p])
            seen.add(page)
            want, scale = P.bounds(case, r, p, c + n)
            assert torch.equal(codes[page].cpu().to(F), want) and torch.equal(scales[page].cpu(), scale)
            assert torch.equal(low[page + 1].cpu(), (want[:, 0].float() * scale[:, None])) and torch.equal(high[page + 1].cpu(), (want[:, 1].float() * scale[:, None]))
    for page in set(range(codes.shape[0])) - seen:
        assert bool((codes[page] == 99).all()) and bool((scales[page] == -5.0).all())


def test_bounds_of_a_step():
    """Only the pages of the step's tokens change, and to what all tokens at once give."""
    case = Paged([(60, 10), (130, 1), (0, 3), (64, 64)], 2, 2, 64, seed=5)
    whole = make_bounds(case)
    codes, scales = K().page_bounds_pool(case.k.shape[0], 2, 64, DEV)
    K().page_bounds(case.k.to(DEV), codes, scales, case.table.to(DEV), ints(case.start), ints(case.pos0), case.max_new)
    touched = {int(case.table[r, p]) for r, (c, n) in enumerate(case.rows) for p in range(c // PAGE, -(-(c + n) // PAGE))}
    for page in range(case.k.shape[0]):
        if page in touched:
            assert torch.equal(codes[page], whole[0][page]) and torch.equal(scales[page], whole[1][page])
        else:
            assert bool((codes[page] == 0).all()) and bool((scales[page] == 0).all())


def test_bounds_of_odd_keys():
    """Keys of zero, the smallest and the largest, ones that are not finite."""
    case = Paged([(0, 64), (0, 64), (0, 64), (0, 64), (0, 7)], 1, 1, 64, seed=6)
    page = [int(case.table[r, 0]) for r in range(5)]
    case.k[page[0]] = 0.0
    case.k[page[1]] = 2.0 ** -130
    case.k[page[1], 0, 3, 5] = 3.3895e38
    case.k[page[2], 0, 9, 9] = math.inf
    case.k[page[3], 0, 1, 2] = math.nan
    codes, scales = make_bounds(case)
    for r in (0, 1, 4):
        want, scale = P.bounds(case, r, 0, case.rows[r][1])
        assert torch.equal(codes[page[r]].cpu().to(F), want) and torch.equal(scales[page[r]].cpu(), scale)
    for r in (2, 3):
        assert bool((codes[page[r]] == 0).all()) and bool(torch.isinf(scales[page[r]]).all())


def select(case, codes, scales, count, first, last, table=None, **kw):
    return K().page_select(case.q.to(DEV), codes, scales, (case.table if table is None else table).to(DEV), ints(case.tok_pos), ints(case.tok_seq), count, case.h, case.g,
                           case.d, first=first, last=last, **kw)


def run_listed(case, pages, ws=None, table=None, scale=None):
    y = K().attn_pages(case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), (case.table if table is None else table).to(DEV), ints(case.tok_pos), ints(case.tok_seq), pages,
                       case.h, case.g, case.d, scale=case.d ** -0.5 if scale is None else scale, workspace=ws)
    torch.cuda.synchronize()
    K().check_status()
    return y


@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("rows,count,first,last", [
    ([(0, 1)], 3, 1, 1),
    ([(700, 1), (64, 1), (63, 2)], 4, 1, 2),
    ([(2000, 3), (130, 1)], 7, 0, 1),
    ([(900, 1), (900, 1)], 1, 1, 1),                        # fewer than must be: the lowest
    ([(1500, 2)], 40, 2, 3),                                # more than there are
])
def test_chosen_pages(heads, kv_heads, d, rows, count, first, last):
    case = Paged(rows, heads, kv_heads, d, seed=count + d)
    codes, scales = make_bounds(case)
    pages = select(case, codes, scales, count, first, last)
    want = [P.choose(case, codes.cpu(), scales.cpu(), t, count, first, last) for t in range(len(case.tok_pos))]
    assert pages.tolist() == want
    y, size = P.listed(case, want, d ** -0.5)
    assert P.off(run_listed(case, pages, ws=workspace()), y, size) <= 1.0


def test_all_pages_are_dense_attention():
    case = Paged([(900, 2), (64, 1), (10, 1)], 8, 2, 128, seed=8)
    codes, scales = make_bounds(case)
    pages = select(case, codes, scales, 20, 1, 1)
    want, size = P.shared(case, 128 ** -0.5)
    assert P.off(run_listed(case, pages, ws=workspace()), want, size) <= 1.0


def test_equal_scores_go_to_the_lower_page():
    case = Paged([(40 * PAGE, 1)], 2, 1, 64, seed=9)
    pages = case.table[0].tolist()
    for p in range(40):                                     # all pages alike
        case.k[pages[p]] = case.k[pages[0]]
    codes, scales = make_bounds(case)
    assert select(case, codes, scales, 9, 0, 1).tolist() == [[[0, 1, 2, 3, 4, 5, 6, 7, 40]]]
    case.q[:] = 0.0                                         # and so are zero queries'
    assert select(case, codes, scales, 9, 2, 2).tolist() == [[[0, 1, 2, 3, 4, 5, 6, 39, 40]]]


def test_pages_that_are_not_there():
    case = Paged([(20 * PAGE + 3, 1), (6 * PAGE, 1)], 4, 2, 64, seed=10)
    codes, scales = make_bounds(case)
    case.table[0, 4] = case.table[0, 20] = -1
    case.table[1, 0] = case.k.shape[0] + 7
    table = case.table.clone()
    case.table[1, 0] = -1
    pages = select(case, codes, scales, 6, 1, 1, table=table)
    want = [P.choose(case, codes.cpu(), scales.cpu(), t, 6, 1, 1) for t in range(2)]
    assert pages.tolist() == want
    y, size = P.listed(case, want, 0.125)
    assert P.off(run_listed(case, pages, ws=workspace(), table=table), y, size) <= 1.0
    y, size = P.shared(case, 0.125)
    assert P.off(run_shared(case, groups=None), y, size) <= 1.0


def test_pages_that_are_not_there_among_shared_ones():
    case = Paged([(9 * PAGE + 5, 1), (9 * PAGE, 2), (9 * PAGE + 70, 1)], 4, 2, 128, share=share([(3, 9)]), seed=11)
    for missing in (0, 3, 8):
        case.table[:, missing] = -1
    y, size = P.shared(case, 0.1)
    assert P.off(run_shared(case, scale=0.1), y, size) <= 1.0


def test_pages_whose_keys_are_not_finite_come_first():
    case = Paged([(30 * PAGE, 1)], 4, 2, 128, seed=12)
    case.k[int(case.table[0, 17]), 1, 5, 5] = math.nan
    codes, scales = make_bounds(case)
    pages = select(case, codes, scales, 3, 1, 1).tolist()
    assert pages == [P.choose(case, codes.cpu(), scales.cpu(), 0, 3, 1, 1)] and 17 in pages[0][1] and 17 not in pages[0][0]


def test_lists_by_hand():
    """Any order, pages twice, holes, pages beyond the token's."""
    case = Paged([(400, 2), (70, 1)], 4, 2, 64, seed=13)
    lists = [[[5, 0, 3, -1, 3], [6, 6, 100, 2, -7]], [[-1, -1, -1, -1, -1], [1, 2, 3, 4, 5]], [[1, 0, 0, 0, 0], [-1, 1, 0, 0, 0]]]
    y, size = P.listed(case, lists, 0.125)
    got = run_listed(case, ints(lists), ws=workspace())
    assert P.off(got, y, size) <= 1.0
    assert bool((got[1, :128] == 0).all())                  # the list that names nothing


# ---- hidden places -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (8, 2, 128), (32, 1, 128)])
def test_values_of_later_tokens_do_not_reach_earlier_ones(heads, kv_heads, d):
    """The step's second token has values that are not finite: those before it stay as they are, those that see it take them."""
    case = Paged([(60, 5), (100, 4)], heads, kv_heads, d, seed=14)
    want, size = P.shared(case, d ** -0.5)
    page, place = int(case.table[0, 0]), 61
    case.v[page, :, place, 3] = math.nan
    case.v[int(case.table[1, 1]), :, 38, 7] = math.inf
    got = run_shared(case, groups=None, ws=workspace())
    for t, bad in ((0, False), (1, True), (4, True), (5, False), (6, False), (7, True), (8, True)):
        feature = 3 if t < 5 else 7
        x = got[t].view(heads, d)
        rest = [i for i in range(d) if i != feature]
        assert bool(torch.isfinite(x[:, feature]).all()) != bad
        w, s = want[t].view(heads, d), size[t].view(heads, d)
        assert P.off(x[:, rest], w[:, rest], s[:, rest]) <= 1.0
        if not bad:
            assert P.off(x, w, s) <= 1.0


def test_queries_before_everything():
    case = Paged([(0, 2), (10, 1)], 4, 2, 64, seed=15)
    case.pos0[0] = -1
    case.tok_pos[:2] = [-1, 0]
    want, size = P.shared(case, 0.125)
    got = run_shared(case, groups=None)
    assert P.off(got, want, size) <= 1.0 and bool((got[0] == 0).all())
    got = run_listed(case, ints([[[0], [0]]] * 3))
    assert bool((got[0] == 0).all()) and bool((got[1] != 0).any())


def test_large_scores():
    case = Paged([(500, 1), (3 * PAGE + 9, 2)], 4, 2, 128, seed=16, k_scale=30.0)
    want, size = P.shared(case, 1.0)                        # scores of some thousands: float32 sums are off by up to 2^-24 of 128 products of 100 each, twice over
    got = run_shared(case, groups=None, scale=1.0)
    assert bool(torch.isfinite(got).all())
    assert float((got.cpu().to(F) - want).abs().max()) <= float(want.abs().max()) * 0.02


# ---- calls ---------------------------------------------------------------------------------------------------------------------------------

def test_strided_queries_and_given_outputs():
    case = Paged([(300, 2), (40, 1)], 4, 2, 64, share=None, seed=17)
    wide = torch.randn(3, 4 * 64 + 2 * 2 * 64, device=DEV).bfloat16()
    wide[:, :256] = case.q.to(DEV)
    out = torch.full((3, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    want = run_shared(case, groups=None)
    got = run_shared(case, groups=None, q=wide[:, :256], out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


def test_tokens_behind_the_last_row_are_left_as_they_were():
    case = Paged([(300, 2), (40, 1)], 4, 2, 64, seed=18)
    want = run_shared(case, groups=None)
    q = torch.cat([case.q, torch.full((4, 256), math.nan, dtype=torch.bfloat16)]).to(DEV)
    out = torch.full((7, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    got = run_shared(case, groups=None, q=q, out=out)
    assert torch.equal(got[:3], want) and bool((got[3:] == 7.0).all())


def test_groups_that_are_none():
    """Overlapping groups, ones beyond the rows, of no rows, of no pages, of more pages than the table has."""
    case = Paged([(4 * PAGE + 7 * i, 1) for i in range(6)], 4, 2, 64, share=share([(4, 4)], 2), seed=19)
    want, size = P.shared(case, 0.125)
    for groups in ([[0, 4, 4], [2, 3, 4]], [[0, 4, 4], [9, 2, 1]], [[0, 0, 4], [0, 2, 4], [2, 2, 4]], [[0, 4, 0]], [[-3, 2, 4], [1, 2, 4]], []):
        assert P.off(run_shared(case, groups=groups), want, size) <= 1.0, groups


def test_many_groups():
    n = 256
    case = Paged([(PAGE + i % 3, 1) for i in range(2 * n)], 2, 1, 64, share=[(i // 2, 1) for i in range(2 * n)], seed=20)
    want, size = P.shared(case, 0.125)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


def test_more_items_than_a_launch_takes():
    case = Paged([(i % 70, 1) for i in range(2500)], 2, 2, 64, seed=21)
    want, size = P.shared(case, 0.125)
    assert P.off(run_shared(case, groups=None, ws=workspace()), want, size) <= 1.0
    lists = [[[0, 1], [1, 0]]] * 2500                        # (tokens of the first page look at the first entry only: nothing, for the second head)
    want, size = P.listed(case, lists, 0.125)
    assert P.off(run_listed(case, ints(lists), ws=workspace()), want, size) <= 1.0


def test_one_workspace_for_calls_one_behind_the_other():
    ws = workspace()
    a = Paged([(200 * PAGE + 5, 1)] * 3, 8, 2, 128, share=share([(3, 200)]), seed=22)
    b = Paged([(3000, 1), (10, 2)], 4, 4, 64, seed=23)
    first, second = run_shared(a), run_shared(b, groups=None)
    for _ in range(3):
        assert torch.equal(run_shared(a, ws=ws), first) and torch.equal(run_shared(b, groups=None, ws=ws), second)


def test_replayed_from_a_graph_with_other_lengths():
    """Everything that a step needs is in device memory: a recorded call goes on with later positions and other groups."""
    case = Paged([(5 * PAGE + i, 1) for i in (0, 30, 63)] + [(100, 1)], 4, 2, 128, share=share([(3, 5)], 1), seed=24)
    ws = workspace()
    codes, scales = make_bounds(case)
    q, k, v, table = case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), wide(case, case.table.to(DEV))
    start, pos0, groups = ints(case.start), ints([0] * 4), ints([[0, 0, 0]])
    pos, seq = ints([0] * 4), ints(case.tok_seq)

    def step():
        y = K().attn_shared(q, k, v, table, start, pos0, groups, 1, 4, 2, 128, scale=0.1, workspace=ws)
        pages = K().page_select(q, codes, scales, table, pos, seq, 3, 4, 2, 128)
        return y, pages, K().attn_pages(q, k, v, table, pos, seq, pages, 4, 2, 128, scale=0.1, workspace=ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, pages, z = step()
    for at, g in ((case.pos0, case.groups[0]), ([5 * PAGE, 5 * PAGE, 5 * PAGE + 2, 3], [0, 3, 5]), ([9, 70, 200, 64], [0, 0, 0])):
        pos0.copy_(ints(at))
        pos.copy_(ints(at))
        groups.copy_(ints([g]))
        graph.replay()
        torch.cuda.synchronize()
        K().check_status()
        case.pos0 = case.tok_pos = list(at)
        want, size = P.shared(case, 0.1)
        assert P.off(y, want, size) <= 1.0
        chosen = [P.choose(case, codes.cpu(), scales.cpu(), t, 3, 1, 1) for t in range(4)]
        assert pages.tolist() == chosen
        want, size = P.listed(case, chosen, 0.1)
        assert P.off(z, want, size) <= 1.0


def test_on_another_stream():
    case = Paged([(2000, 1), (640, 3)], 8, 2, 64, seed=25)
    want = run_shared(case, groups=None)
    q, k, v, table, start, pos0 = case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), case.table.to(DEV), ints(case.start), ints(case.pos0)
    ws = workspace()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = K().attn_shared(q, k, v, table, start, pos0, None, 3, 8, 2, 64, scale=0.125, workspace=ws)
    s.synchronize()
    assert torch.equal(got, want)


def test_two_graphs_over_one_workspace():
    """Recorded one by one, replayed in turn: what one leaves in the scratch memory is nothing to the other."""
    ws = workspace()
    ws.reserve(1 << 22)
    a = Paged([(40 * PAGE + 5 * i, 1) for i in range(6)], 8, 2, 128, share=share([(6, 40)]), seed=31)
    b = Paged([(900, 2), (64, 1), (5 * PAGE, 1)], 4, 4, 64, share=share([(1, 5)], 2), seed=32)
    lists = torch.tensor([[[p for p in (0, 3, 9, -1)]] * 2] * 6, dtype=torch.int32, device=DEV)
    graphs = []
    for case in (a, b):
        q, k, v, table = case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), wide(case, case.table.to(DEV))
        start, pos0, groups, pos, seq = ints(case.start), ints(case.pos0), ints(case.groups).view(-1, 3), ints(case.tok_pos), ints(case.tok_seq)

        def step(case=case, q=q, k=k, v=v, table=table, start=start, pos0=pos0, groups=groups, pos=pos, seq=seq):
            y = K().attn_shared(q, k, v, table, start, pos0, groups, case.max_new, case.h, case.g, case.d, scale=0.1, workspace=ws)
            return y, K().attn_pages(q, k, v, table, pos, seq, lists, 8, 2, 128, scale=0.1, workspace=ws) if case is a else y

        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got, want, step))
    for _ in range(3):
        for graph, got, _, _ in graphs:
            for t in got:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        K().check_status()
        assert all(torch.equal(x, y) for _, got, want, _ in graphs for x, y in zip(got, want))


def test_two_streams_at_once():
    """Two calls at a time, each with a workspace of its own, over one cache."""
    case = Paged([(70 * PAGE + 3 * i, 1) for i in range(12)], 16, 2, 64, share=share([(12, 70)]), seed=33)
    want = run_shared(case)
    q, k, v, table = case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), wide(case, case.table.to(DEV))
    start, pos0, groups = ints(case.start), ints(case.pos0), ints(case.groups)
    streams, spaces = [torch.cuda.Stream() for _ in range(2)], [workspace() for _ in range(2)]
    for ws in spaces:
        ws.reserve(1 << 22)
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, ws in zip(streams, spaces):
            with torch.cuda.stream(s):
                got.append(K().attn_shared(q, k, v, table, start, pos0, groups, 1, 16, 2, 64, scale=0.125, workspace=ws))
    torch.cuda.synchronize()
    K().check_status()
    assert all(torch.equal(y, want) for y in got)
