"""The 4-bit cache's attention in both of its forms, walking the codes and unpacking the rows' pages, on the same inputs: which of them a call takes
is a matter of time and must not show in its results.

Tolerances are test_cache4_gpu.py's (``Case.check``): the result is rounded to bfloat16, the terms to fp16, in the unpacked form keys, values and
queries to fp16 as well, after a power of two that brings a row's largest near fp16's: 2^-7 of the largest value and what rounded keys move."""
import math

import pytest
import torch

from plain_lowbit import attend, rounded4
from test_cache4_gpu import DEV, Case, K, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["codes", "unpacked"])
def way(request, monkeypatch):
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: request.param)
    return request.param


def refilled(c, f):
    """The case's keys and values times f, a number or one for each key/value head, and its queries as they are."""
    g, d = c.g, c.d
    kv = c.qkv[:, c.h * d:].float().view(-1, 2, g, d) * torch.as_tensor(f, device=DEV).view(-1, 1)
    qkv = torch.cat([c.qkv[:, :c.h * d], kv.reshape(-1, 2 * g * d).bfloat16()], 1)
    lens = [a + n for a, n in c.rows]
    K().kv4_store(qkv, None, ints([p for L in lens for p in range(L)]), ints([r for r, L in enumerate(lens) for _ in range(L)]), c.table, c.pool, c.h, g, d)
    at = 0
    for r, L in enumerate(lens):
        x = qkv[at:at + L, c.h * d:].cpu().view(L, 2, g, d)
        c.k[r], c.v[r] = rounded4(x[:, 0]), rounded4(x[:, 1])
        at += L


# ---- pages that are not there ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (16, 2, 64), (8, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("window", [0, 300])
def test_pages_that_are_missing_are_left_out(way, heads, kv_heads, d, window):
    c = Case([(420, 100), (130, 30)], heads, kv_heads, d, seed=21)
    c.table[0, 1:3], c.table[0, 5], c.table[1, 0] = -1, 10 ** 6, -1          # no page, and a number beyond the pool
    gone = [set(range(64, 192)) | set(range(320, 384)), set(range(64))]
    out, at = c.run(window).double().cpu().view(-1, heads, d), 0
    for r, (ctx, n) in enumerate(c.rows):
        for i in (0, 1, n - 1):
            want = attend(c.q[at + i:at + i + 1].cpu().view(1, heads, d), c.k[r], c.v[r], ctx + i, d ** -0.5, window, hidden_keys=gone[r])[0]
            assert float((out[at + i] - want).abs().max()) <= 2.0 ** -7 * float(c.v[r].abs().max()), (r, i)
        at += n


@pytest.mark.parametrize("d,new", [(64, 90), (128, 90), (64, 150), (128, 150)])
def test_rows_without_pages_get_zeros(way, d, new):
    c = Case([(40, new), (40, new)], 4, 2, d, seed=6)
    c.table[0] = -1
    out = c.run().view(2, new, -1)
    assert bool((out[0] == 0).all()) and bool((out[1] != 0).any())
    K().check_status()


@pytest.mark.parametrize("new", [70, 150])
@pytest.mark.parametrize("window", [0, 100])
def test_rows_longer_than_their_table(way, new, window):
    """Places beyond the table's width are not there."""
    c = Case([(200, new), (60, new)], 8, 2, 128, seed=22)
    c.table = c.table[:, :3].contiguous()
    out, at = c.run(window).double().cpu().view(-1, 8, 128), 0
    for r, (ctx, n) in enumerate(c.rows):
        for i in (0, n - 1):
            want = attend(c.q[at + i:at + i + 1].cpu().view(1, 8, 128), c.k[r], c.v[r], ctx + i, 128 ** -0.5, window, hidden_keys=set(range(192, 500)))[0]
            assert float((out[at + i] - want).abs().max()) <= 2.0 ** -7 * float(c.v[r].abs().max()), (r, i)
        at += n
    K().check_status()


@pytest.mark.parametrize("first", [-1, -64, -200])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128)])
def test_queries_before_the_first_position_get_zeros(way, first, heads, kv_heads, d):
    c = Case([(0, 140), (10, 20)], heads, kv_heads, d, seed=23)
    c.pos0[0] = first
    c.max_len = 140
    out = c.run().double().cpu().view(-1, heads, d)
    n = min(140, -first)
    assert bool((out[:n] == 0).all())
    if n < 140:
        want = attend(c.q[n:n + 1].cpu().view(1, heads, d), c.k[0], c.v[0], 0, d ** -0.5)[0]
        assert float((out[n] - want).abs().max()) <= 2.0 ** -7 * float(c.v[0].abs().max())
    K().check_status()


# ---- sizes ----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("exponent", [-60, -30, -22, -18, -12, 0, 12, 20, 60])
@pytest.mark.parametrize("d,new", [(64, 70), (128, 150)])
def test_sizes(way, exponent, d, new):
    """Powers of two in q and in k and v move nothing but the result's size (k up, q down: the same scores)."""
    c = Case([(90, new), (33, 20)], 4, 2, d, seed=11)
    base = c.run()
    f = 2.0 ** exponent
    refilled(c, f)
    out = c.run(q=(c.q.float() / f).bfloat16())
    assert float((out.double() / f - base.double()).abs().max()) <= 2.0 ** -7 * max(float(v.abs().max()) for v in c.v) / f


@pytest.mark.parametrize("d,new", [(64, 70), (128, 150)])
def test_values_of_rows_and_heads_differ_in_size(way, d, new):
    """A head's values 2^-25, its neighbour's 2^18: each result is as good as its own values allow."""
    c = Case([(90, new), (33, 20)], 4, 2, d, seed=24, q_scale=2.0 ** -10)
    refilled(c, [2.0 ** -25, 2.0 ** 18])
    out, at = c.run().double().cpu().view(-1, 4, d), 0
    for r, (ctx, n) in enumerate(c.rows):
        for i in (0, n - 1):
            q = c.q[at + i:at + i + 1].cpu().view(1, 4, d)
            want = attend(q, c.k[r], c.v[r], ctx + i, d ** -0.5)[0]
            for g in range(2):
                moved = 2.0 ** -12 * d ** -0.5 * float(q[0, 2 * g:2 * g + 2].double().norm(dim=-1).max() * c.k[r][:, g].norm(dim=-1).max())
                err = float((out[at + i, 2 * g:2 * g + 2] - want[2 * g:2 * g + 2]).abs().max())
                assert err <= (2.0 ** -7 + 2 * moved) * float(c.v[r][:, g].abs().max()), (r, i, g)
        at += n


# ---- scratch memory -------------------------------------------------------------------------------------------------------------

def peak(f):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("window", [0, 200])
def test_scratch_is_of_the_pages_that_are_seen(window):
    """A long prompt among short ones, with the rows' lengths known on the host: copies of the pages that each row sees, not of as many as the longest
    has; and the same bits without the lengths."""
    rows = [(0, 6000)] + [(0, 200)] * 31
    c = Case(rows, 8, 8, 64, seed=25)
    c.row_lens = rows
    known, took = peak(lambda: c.run(window, row_lens=rows))
    pages = sum(-(-n // 64) for _, n in rows)
    copies, queries = pages * 8 * 64 * 64 * 4, 2 * c.q.numel()
    assert took <= copies + 2 * queries + (4 << 20), (took, copies)                 # the queries' copies, the result, the plan
    assert torch.equal(c.run(window), known)
    c.check(known, window, only=(0, 63, 64, 199, 4000, 5999))


@pytest.mark.parametrize("heads,kv_heads,d,window", [(4, 4, 64, 0), (40, 20, 64, 90), (8, 2, 128, 0), (7, 1, 128, 150)])
@pytest.mark.parametrize("known", [True, False])
def test_rows_in_several_passes(heads, kv_heads, d, window, known, monkeypatch):
    """As many passes as two of the longest rows' pages at a time make of it: the same bits as in one."""
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: False)
    rows = [(300, 200), (0, 130), (0, 0), (700, 17), (64, 64), (5, 300), (0, 1), (600, 129), (130, 40)]
    c = Case(rows, heads, kv_heads, d, seed=26)
    c.table[1, 0], c.table[7, 9] = -1, -1
    kw = dict(row_lens=rows) if known else {}
    one = c.run(window, **kw)
    monkeypatch.setattr(K(), "KV4_PROMPT_BYTES", 0)
    assert torch.equal(c.run(window, **kw), one)
    K().check_status()


@pytest.mark.parametrize("said", [dict(max_len=100), dict(row_lens=[(90, 60), (0, 10)]), dict(row_lens=[(0, 1), (0, 1)])])
def test_rows_longer_than_was_said(said, monkeypatch):
    """What is beyond the sizes of the call is hidden; nothing is written or read out of place (the rows before stay right)."""
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: False)
    c = Case([(90, 60), (200, 150)], 4, 2, 64, seed=27)
    want = c.run().view(210, 4, 64)
    lens = said.pop("row_lens", None)
    c.max_len = said.get("max_len", c.max_len)
    out = c.run(row_lens=lens).view(210, 4, 64)
    assert bool(out.isfinite().all())
    if lens is None or lens[0] == (90, 60):
        assert torch.equal(out[:10], want[:10])                                     # positions 90 .. 99, all of whose keys are within the sizes
    K().check_status()


def test_row_lens_of_another_number_of_rows_are_refused():
    from exl3_server_b200.ops.lib import KernelLibraryError
    c = Case([(90, 60)], 4, 2, 64, seed=28)
    with pytest.raises(KernelLibraryError, match="row_lens"):
        c.run(row_lens=[(90, 60), (0, 1)])


# ---- rows of a few tokens beside prompts ----------------------------------------------------------------------------------------

MIXED = [(700, 1), (0, 200), (1300, 1), (64, 1), (90, 150), (0, 1), (0, 0), (513, 2), (40, 17)]


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (16, 2, 64), (40, 1, 64), (8, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("beside", [True, False])
def test_single_tokens_beside_prompts(heads, kv_heads, d, window, known, beside, monkeypatch):
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: False)
    monkeypatch.setattr(K(), "KV4_BESIDE_US", 0.0 if beside else 1e9)
    c = Case(MIXED, heads, kv_heads, d, seed=29)
    out = c.run(window, row_lens=MIXED if known else None, out=torch.full_like(c.q, math.nan))
    c.check(out, window, only=(0, 1, 16, 149, 199))
    K().check_status()


def test_single_tokens_beside_a_prompt_are_not_unpacked():
    """Long rows that decode beside a short prompt take no scratch for their pages, with or without the lengths."""
    rows = [(6000, 1)] * 15 + [(0, 300)]
    c = Case(rows, 8, 2, 128, seed=30)
    for lens in (rows, None):
        _, took = peak(lambda: c.run(row_lens=lens))
        one = 95 * 2 * 64 * 128 * 4                                    # copies of a long row's pages
        chunks = 16 * 8 * 24 * 132 * 4 * 4                             # records of up to 24 chunks of 8 heads, 16 columns at most
        assert took <= (0 if lens else 16) * one + 4 * 2 * c.q.numel() + chunks + (4 << 20), took
    c.check(c.run(row_lens=rows), only=(0, 299))


@pytest.mark.parametrize("heads,kv_heads", [(32, 1), (34, 2), (16, 16)])
def test_one_token_a_row_without_starts(heads, kv_heads, monkeypatch):
    """``row_start`` None goes with tiles too, and with more query heads a key/value head than 16."""
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: False)
    c = Case([(100, 1), (9, 1)], heads, kv_heads, 128, seed=5)
    want = c.run(tiles=False)
    c.check(want)
    assert torch.equal(K().kv4_attn(c.q, c.pool, c.table, None, c.pos0, c.tiles, 1, c.max_len, heads, kv_heads, 128, 128 ** -0.5), want)


# ---- arguments ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
@pytest.mark.parametrize("d,new", [(64, 70), (128, 150)])
def test_scales(way, scale, d, new):
    """Any finite scale: a negative one turns the order round, 0 gives the mean of what a query sees."""
    c = Case([(90, new)], 4, 2, d, seed=31)
    out = K().kv4_attn(c.q, c.pool, c.table, c.start, c.pos0, c.tiles, c.max_new, c.max_len, 4, 2, d, scale).double().cpu().view(new, 4, d)
    for i in (0, 3, new - 1):
        q = c.q[i:i + 1].cpu().view(1, 4, d)
        want = attend(q, c.k[0], c.v[0], 90 + i, scale)[0]
        moved = 2.0 ** -12 * abs(scale) * float(q.double().norm(dim=-1).max() * c.k[0].norm(dim=-1).max())
        assert float((out[i] - want).abs().max()) <= (2.0 ** -7 + 2 * moved) * float(c.v[0].abs().max())


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_scales_that_are_not_finite_are_refused(way, scale):
    from exl3_server_b200.ops.lib import KernelLibraryError
    c = Case([(90, 70)], 4, 2, 64, seed=31)
    with pytest.raises(KernelLibraryError, match="scale"):
        K().kv4_attn(c.q, c.pool, c.table, c.start, c.pos0, c.tiles, c.max_new, c.max_len, 4, 2, 64, scale)


def test_one_token_of_a_matrix_with_any_stride():
    """A step of one token has no distance between tokens, whatever the stride says."""
    k = K()
    c = Case([(10, 1)], 4, 2, 64, seed=14)
    want = c.run()
    odd = torch.zeros(1, 8 * 64 + 5, device=DEV).bfloat16()
    odd[:, :512] = c.qkv[10:11]
    odd[:, :256] = c.q
    pool = c.pool.clone()
    q = k.kv4_store(odd[:, :512], None, ints([10]), ints([0]), c.table, pool, 4, 2, 64)
    assert torch.equal(q, c.q) and torch.equal(pool, c.pool) and torch.equal(c.run(q=odd[:, :256]), want)


def test_lists_of_tiles_that_are_refused():
    from exl3_server_b200.ops.lib import KernelLibraryError
    c = Case([(90, 200)], 4, 2, 64, seed=32)
    a, b, n = c.tiles
    for tiles in ((a.long(), b, n), (a, b.long(), n), (a[:1], b, n), (a, b, n + 1)):
        c.tiles = tiles
        with pytest.raises(KernelLibraryError, match="tiles"):
            c.run()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("first", [-3, 40])
def test_windows_beyond_every_key(way, window, first):
    c = Case([(40, 100)], 8, 2, 64, seed=33)
    c.pos0[0] = first
    assert torch.equal(c.run(window), c.run(0))


# ---- what must not matter, in both forms ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("new,window", [(90, 0), (90, 30), (150, 0), (150, 30)])
def test_what_lies_in_unused_places_does_not_matter(way, heads, kv_heads, d, new, window):
    """Places behind the last token, and before the window, hold keys and values of 1e30, then NaN."""
    c = Case([(100, new)], heads, kv_heads, d, seed=16)
    want = c.run(window)
    width = (heads + 2 * kv_heads) * d
    places = list(range(100 + new, c.table.shape[1] * 64)) + (list(range(0, 100 - 30 + 1)) if window else [])
    for filler in (torch.randn(len(places), width, device=DEV) * 1e30, torch.full((len(places), width), math.nan, device=DEV)):
        K().kv4_store(filler.bfloat16(), None, ints(places), ints([0] * len(places)), c.table, c.pool, heads, kv_heads, d)
        assert torch.equal(c.run(window), want)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d,new", [(64, 80), (128, 150)])
def test_queries_that_are_not_finite(way, value, d, new):
    c = Case([(70, new)], 4, 2, d, seed=10)
    q = c.q.clone()
    q[0, d + 6] = value                                                 # head 1 of the first token
    out = c.run(q=q).view(new, 4, d)
    assert bool(out[0, 1].isnan().all()) and bool(out[0, [0, 2, 3]].isfinite().all()) and bool(out[1:].isfinite().all())


def test_steps_in_a_row_in_one_workspace():
    """Steps of other rows, lengths and head sizes, launched one behind the other into the same scratch memory: each as it is alone."""
    from exl3_server_b200.engine.batch import Workspace
    sets = [([(300, 200), (0, 130), (700, 17)], 8, 2, 128, 0), ([(0, 700)], 4, 4, 64, 0), ([(64, 300), (5, 150), (900, 1), (0, 140)], 8, 2, 128, 100),
            ([(0, 140)] * 9, 16, 16, 64, 0), ([(20, 150), (0, 400)], 7, 1, 128, 0)]
    cases = [(Case(rows, h, g, d, seed=40 + i), window, rows) for i, (rows, h, g, d, window) in enumerate(sets)]
    cases[0][0].table[1, 0] = -1
    want = []
    for c, window, rows in cases:
        want.append(c.run(window, workspace=Workspace(torch.device(DEV)), row_lens=rows))
        torch.cuda.synchronize()
    ws = Workspace(torch.device(DEV))
    for turn in range(12):
        order = [(3 * turn + i) % 5 for i in range(5)]
        got = [(i, cases[i][0].run(cases[i][1], workspace=ws, row_lens=cases[i][2] if turn % 2 else None)) for i in order + order[::2]]
        assert all(torch.equal(out, want[i]) for i, out in got), turn
    K().check_status()


def test_a_workspace_grows_in_place_of_what_it_was():
    """The smaller buffer is given back before the larger one is made, unless recorded graphs may hold its address."""
    from exl3_server_b200.engine.batch import Workspace
    n = 40 << 20
    for keep in (False, True):
        torch.cuda.empty_cache()
        ws = Workspace(torch.device(DEV), keep_outgrown=keep)
        first = ws.plain(n).data_ptr()
        _, took = peak(lambda: ws.plain(2 * n) is None)
        assert (took <= 4 * n + (1 << 20)) == (not keep), took      # from n floats to 2 n: n more, 2 n where both are held
        assert not keep or ws._outgrown[0].data_ptr() + 4 * Workspace.COUNTERS == first
        del ws
