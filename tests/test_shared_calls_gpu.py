"""Calls of attention over shared and over chosen pages that the tests of their results do not make: at the limits of what the kernels take, with arrays that are laid out otherwise, and what
they write into beside the output."""
import math

import pytest
import torch

import plain_pages as P
import test_shared_pages_gpu as base
from plain_pages import PAGE, Paged
from test_shared_pages_gpu import DEV, K, ints, run_shared, share, wide, workspace

pytestmark = pytest.mark.gpu


class Guarded:
    """A workspace whose buffer ends where the call's scratch memory does, with a pattern behind it."""

    GUARD = 16 << 20      # floats

    def __init__(self):
        self.buf, self.asked = None, 0

    def floats(self, n):
        self.asked = n
        self.buf = torch.zeros(n + self.GUARD, dtype=torch.float32, device=DEV)
        self.buf[n:] = 7.0
        return self.buf[:n]

    def untouched(self):
        return bool((self.buf[self.asked:] == 7.0).all()) and bool((self.buf[:65536].view(torch.int32) == 0).all())


# ---- scratch memory -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,new,heads,kv_heads,groups", [(300, 5, 16, 1, 32), (300, 10, 8, 1, 30)])
def test_groups_that_are_left_alone_write_no_further_than_their_scratch(rows, new, heads, kv_heads, groups):
    """Without its groups each row has a tile, with them there are too many: the scratch memory is that of the call that is made."""
    cuts = [rows * i // groups for i in range(groups + 1)]
    case = Paged([(PAGE, new)] * rows, heads, kv_heads, 64, share=share([(b - a, 1) for a, b in zip(cuts, cuts[1:])]), seed=40)
    ws = Guarded()
    want, size = P.shared(case, 0.125)
    got = run_shared(case, ws=ws, little=True)
    assert ws.untouched()
    assert P.off(got, want, size) <= 1.0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("groups", [[], [[6 * j, 6, 1] for j in range(33)]])
def test_rows_that_are_not_one_behind_the_other(d, groups):
    """Rows that all claim the same tokens make more tiles than the tokens can: no result is defined, and nothing is written but the output and the scratch memory."""
    k, case = K(), Paged([(3 * PAGE, 100)], 16, 1, d, seed=41)
    T, rows = 100, 200
    out = torch.full((T + 64, 16 * d), 7.0, dtype=torch.bfloat16, device=DEV)
    table = wide(case, case.table.to(DEV)).expand(rows, -1)
    start = ints([0, T] * (rows // 2) + [0])
    ws = Guarded()
    k.attn_shared(case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), table, start, ints([3 * PAGE] * rows), ints(groups).view(-1, 3), 100, 16, 1, d, scale=0.1, workspace=ws, out=out[:T])
    torch.cuda.synchronize()
    k.check_status()
    assert ws.untouched() and bool((out[T:] == 7.0).all())
    want, size = P.shared(case, 0.1)
    assert P.off(run_shared(case, scale=0.1), want, size) <= 1.0


@pytest.mark.parametrize("news", [[1100], [600, 600]])
def test_rows_of_more_tokens_than_said_that_cannot_be_counted(news):
    """Rows bring hundreds of tokens where the call says one each, behind so many pages that their units pass 31 bits (a token's eight queries are an item of
    more than 2^21 - 125 units: 1,025 of them are too many): the status says so, and nothing is written."""
    k, width, T = K(), 1 << 19, sum(news)
    pool = torch.zeros(1, 1, PAGE, 128, dtype=torch.bfloat16, device=DEV)
    q, out = torch.zeros(T, 1024, dtype=torch.bfloat16, device=DEV), torch.full((T, 1024), 7.0, dtype=torch.bfloat16, device=DEV)
    table = torch.full((len(news), width), -1, dtype=torch.int32, device=DEV)
    start, pos0 = ints([sum(news[:i]) for i in range(len(news) + 1)]), ints([width * PAGE - 2000] * len(news))
    ws = Guarded()
    k.attn_shared(q, pool, pool, table, start, pos0, None, 1, 8, 1, 128, scale=0.1, workspace=ws, out=out)
    torch.cuda.synchronize()
    with pytest.raises(K().KernelLibraryError, match="more tokens than max_new"):
        k.check_status()
    assert bool((out == 7.0).all()) and ws.untouched()
    k.check_status()
    case = Paged([(100, 3)], 8, 1, 128, seed=42)            # (fewer than that are answered)
    want, size = P.shared(case, 0.1)
    case.max_new = 1
    assert P.off(run_shared(case, groups=None, scale=0.1), want, size) <= 1.0


# ---- the limits of the tensor cores' list of tiles -----------------------------------------------------------------------------------

@pytest.mark.parametrize("prompts,new", [(20, 50), (22, 50)])
def test_groups_on_both_sides_of_the_most_tiles(prompts, new):
    """1,000 tokens of 128 heads are 500 tiles and 4 groups; 1,100 are 550, which is too many: the rows then read for themselves."""
    shares = share([(prompts // 4, 1 + j) for j in range(4)], prompts - prompts // 4 * 4)
    case = Paged([((s[1] * PAGE if s else 0) + r % 9, new) for r, s in enumerate(shares)], 128, 1, 64, share=shares, seed=43)
    want, size = P.shared(case, 0.125)
    table = torch.cat([case.table, torch.full((prompts, 20 - case.table.shape[1]), -1, dtype=torch.int32)], 1)
    used, _, tiles = K()._shared_plan(148, prompts * new, prompts, 128, 1, 64, 4, new, 20)[1:]
    assert (used, tiles) == ((4, 504) if prompts == 20 else (0, 0))
    case.table = table
    got = run_shared(case, ws=workspace(), little=True)
    assert P.off(got, want, size) <= 1.0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,tiles", [(600, 302), (1020, 512), (1022, 0)])
def test_prompts_on_both_sides_of_the_most_tiles(new, tiles, d):
    """128 heads: two tokens a tile, and one tile more for each row.  Beyond 512 of a key/value head the prompts' queries walk."""
    case = Paged([(70, new - 3), (9, 3)], 128, 1, d, seed=44)
    assert K()._shared_plan(148, new, 2, 128, 1, d, 0, new - 3, case.table.shape[1])[3] == tiles
    want, size = P.shared(case, d ** -0.5)
    assert P.off(run_shared(case, groups=None, ws=workspace()), want, size) <= 1.0


def test_more_new_tokens_allowed_than_there_are():
    """``max_new`` says how many tokens a row may bring, not how many there are."""
    case = Paged([(r % 90, 1) for r in range(1100)], 8, 1, 64, seed=45)
    want, size = P.shared(case, 0.125)
    case.max_new = 1 << 30
    assert P.off(run_shared(case, groups=None, ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("high", ["shared", "own"])
def test_values_that_are_not_finite_behind_keys_of_no_weight(high, d, rows):
    """The rows' own keys are so far below the shared ones (or these below them) that their weight rounds to zero: a value that is not finite is seen all the same, as where rows
    read for themselves.  Few and many queries, which are joined differently."""
    case = Paged([(4 * PAGE + 3, 1)] * rows, 8, 1, d, share=share([(rows, 4)]), seed=46)
    shared, own = case.table[0, :4].long(), case.table[:, 4].long()
    case.q.fill_(1.0)
    case.k[:] = 4.0 if high == "own" else -4.0
    case.k[shared] = -4.0 if high == "own" else 4.0
    case.v[:] = torch.randn(case.v.shape, generator=torch.Generator().manual_seed(1)).bfloat16()
    want, size = P.shared(case, 0.5)                        # scores of d * 2 and -d * 2: weights of e^-256 and less
    if high == "own":
        case.v[shared[1], :, 9, 5] = math.nan
        case.v[shared[2], :, 60, 7] = math.inf
    else:
        case.v[own, :, 1, 5] = math.nan
        case.v[own, :, 3, 7] = math.inf
    rest = [i for i in range(d) if i not in (5, 7)]
    for groups in ("own", None):
        got = run_shared(case, groups=groups, scale=0.5, ws=workspace()).view(rows, 8, d)
        assert not bool(torch.isfinite(got[..., [5, 7]]).any()), groups
        assert P.off(got[..., rest], want.view(rows, 8, d)[..., rest], size.view(rows, 8, d)[..., rest]) <= 1.0


@pytest.mark.parametrize("d", [64, 128])
def test_lists_of_tokens_beyond_the_table(d):
    """As many entries are looked at as the token's position has pages, however wide the table is; pages beyond the table are not there."""
    case = Paged([(200, 1), (3000, 1), (130, 1)], 4, 2, d, seed=47)
    case.table = case.table[:, :4].contiguous()
    case.tok_pos[0] = case.pos0[0] = 1 << 30
    lists = [[[-1, 9, -1, 4, 5, 1, 0], [-1, -1, -1, -1, -1, -1, 3]], [[50, 46, 40, 30, 2, 3, 1], [-1] * 5 + [0, 0]], [[-1, -1, 2, 1, 0, 0, 0], [7, 0, 1, 2, 2, 2, 2]]]
    case.k[case.table[0].long()] = torch.randn(4, 2, PAGE, d, generator=torch.Generator().manual_seed(2)).bfloat16()      # (the whole of row 0's pages is seen)
    case.v[case.table[0].long()] = torch.randn(4, 2, PAGE, d, generator=torch.Generator().manual_seed(3)).bfloat16()
    flat = Paged([(255, 1), (255, 1), (130, 1)], 4, 2, d, seed=47)      # the same rows, as far as the table goes
    flat.table, flat.k, flat.v, flat.q = case.table, case.k, case.v, case.q
    looked = [[[p if 0 <= p < 4 else -1 for p in entries] for entries in token] for token in lists]
    # (the plain form looks at as many entries as pages up to its position: the ones that count, first)
    looked[0], looked[1] = ([sorted(entries, key=lambda p: p < 0) for entries in looked[t]] for t in (0, 1))
    want, size = P.listed(flat, looked, d ** -0.5)
    assert P.off(base.run_listed(case, ints(lists), ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("others", [0, 1100])
def test_positions_far_before_everything(others):
    """A row that begins further below position 0 than its table is long, walked (beside more rows than have tiles) and in tiles: its later tokens see what they see."""
    case = Paged([(0, 100)] + [(0, 0)] * others, 1, 1, 64, seed=48)
    case.table = case.table[:, :1].contiguous()
    case.pos0[0] = -70
    case.tok_pos = list(range(-70, 30))
    want, size = P.shared(case, 0.125)
    got = run_shared(case, groups=None)
    assert P.off(got, want, size) <= 1.0 and bool((got[:70] == 0).all())


# ---- arrays that are laid out otherwise -------------------------------------------------------------------------------------------------

def cut(x, left=8, right=24):
    """The same matrix as part of a wider one."""
    whole = torch.full((x.shape[0], left + x.shape[1] + right), math.nan if x.is_floating_point() else -7, dtype=x.dtype, device=DEV)
    whole[:, left:left + x.shape[1]] = x.to(DEV)
    return whole[:, left:left + x.shape[1]]


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (16, 2, 128), (32, 1, 128)])
@pytest.mark.parametrize("rows,groups", [
    ([(5 * PAGE + 3, 1), (5 * PAGE, 1), (5 * PAGE + 99, 1), (7, 1)], [(3, 5)]),
    ([(PAGE, 90), (PAGE + 70, 130), (300, 2)], [(2, 1)]),
    ([(20, 150), (0, 1)], []),
])
def test_shared_with_strided_queries_and_tables(heads, kv_heads, d, rows, groups):
    case = Paged(rows, heads, kv_heads, d, share=share(groups, len(rows) - sum(n for n, _ in groups)), seed=50)
    want, size = P.shared(case, d ** -0.5)
    table = cut(wide(case, case.table.to(DEV)), 3, 5)
    assert not table.is_contiguous()
    got = K().attn_shared(cut(case.q), case.k.to(DEV), case.v.to(DEV), table, ints(case.start), ints(case.pos0), ints(case.groups).view(-1, 3), case.max_new, heads, kv_heads, d,
                          scale=d ** -0.5, workspace=workspace())
    torch.cuda.synchronize()
    K().check_status()
    assert P.off(got, want, size) <= 1.0


@pytest.mark.parametrize("width", [0, 600, 32768])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (16, 2, 128)])
def test_choice_with_strided_queries_and_wide_tables(heads, kv_heads, d, width):
    """Bounds, choice and attention over a table that is part of a wider one, and as wide as a recorded step's may be."""
    k, case = K(), Paged([(1500, 1), (90, 2), (0, 1)], heads, kv_heads, d, seed=51)
    table = case.table.to(DEV)
    if width:
        table = torch.cat([table, torch.full((3, width - table.shape[1]), -1, dtype=torch.int32, device=DEV)], 1)
    table = cut(table, 3, 5)
    codes, scales = k.page_bounds_pool(case.k.shape[0], kv_heads, d, DEV)
    lens = [c + n for c, n in case.rows]
    k.page_bounds(case.k.to(DEV), codes, scales, table, ints([sum(lens[:i]) for i in range(4)]), ints([0] * 3), max(lens))
    pages = k.page_select(cut(case.q), codes, scales, table, ints(case.tok_pos), ints(case.tok_seq), 5, heads, kv_heads, d, first=1, last=2)
    want = [P.choose(case, codes.cpu(), scales.cpu(), t, 5, 1, 2) for t in range(4)]
    assert pages.tolist() == want
    y = k.attn_pages(cut(case.q), case.k.to(DEV), case.v.to(DEV), table, ints(case.tok_pos), ints(case.tok_seq), pages, heads, kv_heads, d, scale=0.1, workspace=workspace())
    torch.cuda.synchronize()
    k.check_status()
    right, size = P.listed(case, want, 0.1)
    assert P.off(y, right, size) <= 1.0


# ---- more rows than a launch of the walk takes ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new", [1, 3, 33])
def test_groups_among_more_rows_than_a_launch_takes(new):
    """1,200 rows: groups in the first launch, across both and in the second; a row of many tokens has no tile of its own then."""
    groups = share([(300, 2), (400, 1)], 100) + [(9, 1)] * 350 + [None] * 50
    case = Paged([((s[1] * PAGE if s else 0) + r % 9, new if r % 400 == 7 else 1 + r % min(new, 3)) for r, s in enumerate(groups)], 4, 2, 64, share=groups, seed=52)
    want, size = P.shared(case, 0.125)
    assert P.off(run_shared(case, ws=workspace()), want, size) <= 1.0


@pytest.mark.parametrize("new", [1, 70])
def test_tables_so_wide_that_a_launch_takes_few_rows(new):
    """Rows of 2^18 pages for 16 heads of 128: 127 of one token fill 31 bits of units."""
    shares = share([(150, 3)], 20)
    case = Paged([((s[1] * PAGE if s else 0) + r % 9, new if r % 60 == 0 else 1) for r, s in enumerate(shares)], 16, 16, 128, share=shares, seed=53)
    want, size = P.shared(case, 0.1)
    table = case.table
    case.table = torch.full((len(shares), 1 << 18), -1, dtype=torch.int32)
    case.table[:, :table.shape[1]] = table
    for groups in ("own", None):
        assert P.off(run_shared(case, groups=groups, ws=workspace(), scale=0.1, little=True), want, size) <= 1.0
