"""The 4-bit cache's attention in both of its forms, walking the codes and unpacking the rows' pages, on the same inputs: which of them a call takes
is a matter of time and must not show in its results.

Tolerances are test_cache4_gpu.py's (``Case.check``): the result is rounded to bfloat16, the terms to fp16, in the unpacked form keys, values and
queries to fp16 as well: 2^-7 of the largest value and what rounded keys move."""
import pytest
import torch

from plain_lowbit import attend
from test_cache4_gpu import DEV, Case, K, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["codes", "unpacked"])
def way(request, monkeypatch):
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: request.param)
    return request.param


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
