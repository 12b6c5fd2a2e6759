"""The 4-bit cache on the GPU: storing, reading back, attention over it for single tokens, a few and prompts, against plain float64;
what may lie in hidden places; refusals.

Tolerances, fixed before the first run.  Storing without a rotation is exact (the format's float32 steps, restated).  With one, a key may land on the
neighbouring code where its float32 value and the float64 one lie on two sides of a code's edge: fewer than one in a thousand, and never by
more than one step.  Attention: with |v| <= V over what a query sees, the result is rounded to bfloat16 (2^-9 V) and the terms p sc to fp16
(2^-11 of at most 2 V: values stand at most a group's range from their minimum); scores are float32 sums, off by some 1e-6 of |q| |k|: 2^-7 V holds
them all with room.  Prompts round K, V and q to fp16: K moves a score by up to 2^-12 scale |q| |k|, which joins the bound."""
import math

import pytest
import torch

from plain_lowbit import attend, page_values, rotated, rounded4, step4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F = torch.float64


def K():
    from exl3_server_b200.ops import kernels
    return kernels


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Case:
    """Rows with ``ctx`` stored tokens and ``new`` tokens more, on scrambled pages whose every other place holds NaN words."""

    def __init__(self, rows, heads, kv_heads, d, seed=0, spare=2, q_scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        k = K()
        self.rows, self.h, self.g, self.d = rows, heads, kv_heads, d
        pages = [-(-(c + n) // 64) for c, n in rows]
        total = sum(pages) + spare
        order = torch.randperm(total, generator=gen).tolist()
        width = max(pages + [1])
        self.table = torch.full((len(rows), width), -1, dtype=torch.int32)
        for r, n in enumerate(pages):
            self.table[r, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.table = self.table.to(DEV)
        self.pool = torch.full((total, kv_heads, k.kv4_page_bytes(d)), 0xFF, dtype=torch.uint8, device=DEV)
        lens = [c + n for c, n in rows]
        kv = [(torch.randn(L, 2 * kv_heads * d, generator=gen) * torch.exp(0.5 * torch.randn(1, 2 * kv_heads * d, generator=gen))).bfloat16() for L in lens]
        self.qkv = torch.cat([torch.cat([torch.zeros(L, heads * d, dtype=torch.bfloat16), x], 1) for L, x in zip(lens, kv)]).to(DEV)
        pos, seq = ints([p for L in lens for p in range(L)]), ints([r for r, L in enumerate(lens) for _ in range(L)])
        k.kv4_store(self.qkv, None, pos, seq, self.table, self.pool, heads, kv_heads, d)
        self.k = [rounded4(x[:, :kv_heads * d].view(-1, kv_heads, d)) for x in kv]
        self.v = [rounded4(x[:, kv_heads * d:].view(-1, kv_heads, d)) for x in kv]
        new = [n for _, n in rows]
        self.start = ints([sum(new[:i]) for i in range(len(new) + 1)])
        self.pos0 = ints([c for c, _ in rows])
        self.q = (q_scale * torch.randn(sum(new), heads * d, generator=gen)).bfloat16().to(DEV)
        tiles = sorted(((c + min(a + 128, n), r, a) for r, (c, n) in enumerate(rows) for a in range(0, n, 128)), key=lambda t: -t[0])
        self.tiles = (ints([r for _, r, _ in tiles]), ints([a for _, _, a in tiles]), len(tiles))
        self.max_new, self.max_len = max(new + [0]), max(lens + [0])

    def run(self, window=0, tiles=True, workspace=None, q=None, **kw):
        return K().kv4_attn(self.q if q is None else q, self.pool, self.table, self.start, self.pos0, self.tiles if tiles else None, self.max_new,
                            self.max_len, self.h, self.g, self.d, self.d ** -0.5, window=window, workspace=workspace, **kw)

    def check(self, out, window=0, only=None):
        out = out.double().cpu().view(-1, self.h, self.d)
        at = 0
        for r, (c, n) in enumerate(self.rows):
            q = self.q[at:at + n].cpu().view(n, self.h, self.d)
            picked = range(n) if only is None else [i for i in only if i < n]
            for i in picked:
                want = attend(q[i:i + 1], self.k[r], self.v[r], c + i, self.d ** -0.5, window)[0]
                big = self.v[r][:c + i + 1].abs().max()
                moved = 2.0 ** -12 * self.d ** -0.5 * q[i].double().norm(dim=-1).max() * self.k[r][:c + i + 1].norm(dim=-1).max()
                bound = float((2.0 ** -7 + 2 * moved) * big)
                err = float((out[at + i] - want).abs().max())
                assert math.isfinite(err) and err <= bound, (r, i, err, bound)
            at += n


# ---- storing and reading back ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,heads,kv_heads", [(1, 4, 4), (3, 6, 2), (70, 3, 1), (300, 16, 2)])
def test_store_without_rotation_is_exact(d, T, heads, kv_heads):
    k = K()
    g = torch.Generator().manual_seed(T + d)
    wide = (torch.randn(T, (heads + 2 * kv_heads) * d + 16, generator=g) * 3).bfloat16().to(DEV)
    qkv = wide[:, 8:8 + (heads + 2 * kv_heads) * d]                     # rows further apart than they are long
    pages = -(-(T + 61) // 64)
    table = torch.randperm(pages + 2, generator=g)[:pages].to(torch.int32).to(DEV)[None]
    pool = k.kv4_pool(pages + 2, kv_heads, d, DEV)
    pos = torch.arange(61, 61 + T, dtype=torch.int32, device=DEV)        # from the middle of a page on
    q = k.kv4_store(qkv, None, pos, torch.zeros(T, dtype=torch.int32, device=DEV), table, pool, heads, kv_heads, d)
    assert torch.equal(q, qkv[:, :heads * d])
    ko, vo = k.kv4_load(pool, table[0].contiguous(), d)
    x = qkv[:, heads * d:].cpu().view(T, 2, kv_heads, d)
    for got, want in ((ko, x[:, 0]), (vo, x[:, 1])):
        got = got.transpose(1, 2).reshape(-1, kv_heads, d)[61:61 + T].cpu()
        assert torch.equal(got, rounded4(want).float().bfloat16())       # (8 x 4 bits: float32 holds the value, one rounding)
    page = int(table[0, 0])
    kp, vp = page_values(pool[page, kv_heads - 1], d)
    assert torch.equal(ko[0, kv_heads - 1].cpu(), kp.float().bfloat16()) and torch.equal(vo[0, kv_heads - 1].cpu(), vp.float().bfloat16())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", [0, 777, 60000])
def test_store_rotates_as_the_formula(d, first):
    k = K()
    T, heads, kv_heads = 40, 5, 2
    g = torch.Generator().manual_seed(first + d)
    qkv = torch.randn(T, (heads + 2 * kv_heads) * d, generator=g).bfloat16().to(DEV)
    pos = torch.arange(first, first + T, dtype=torch.int32, device=DEV)
    pages = (first + T - 1) // 64 + 1
    table = torch.full((1, pages), -1, dtype=torch.int32, device=DEV)
    lo = first // 64
    table[0, lo:] = torch.arange(pages - lo, dtype=torch.int32, device=DEV)
    pool = k.kv4_pool(pages - lo, kv_heads, d, DEV)
    freq = k.rotary_table(10000.0 ** (-torch.arange(d // 2, dtype=F) / (d // 2))).to(DEV)
    q = k.kv4_store(qkv, freq, pos, torch.zeros(T, dtype=torch.int32, device=DEV), table, pool, heads, kv_heads, d)
    x = qkv.cpu().view(T, heads + 2 * kv_heads, d)
    turned = rotated(x, pos.cpu())
    assert float((q.double().cpu().view(T, heads, d) - turned[:, :heads]).abs().max()) <= 2.0 ** -8 * float(turned.abs().max())
    ko, _ = k.kv4_load(pool, torch.arange(pages - lo, dtype=torch.int32, device=DEV), d)
    got = ko.transpose(1, 2).reshape(-1, kv_heads, d)[first - lo * 64:][:T].double().cpu()
    want = rounded4(turned[:, heads:heads + kv_heads])
    off = (got - want).abs()
    step = step4(turned[:, heads:heads + kv_heads])
    near = off <= 2.0 ** -8 * want.abs() + 1e-6
    assert float((~near).double().mean()) < 1e-3 and bool((off <= 1.1 * step + 2.0 ** -8 * want.abs()).all())


def test_store_leaves_other_tokens_alone_and_skips_places_that_are_not_there():
    k = K()
    d, heads, kv_heads = 64, 2, 2
    pool = torch.randint(0, 255, (4, kv_heads, k.kv4_page_bytes(d)), dtype=torch.uint8, device=DEV)
    before = pool.clone()
    qkv = torch.randn(4, (heads + 2 * kv_heads) * d, device=DEV).bfloat16()
    table = ints([[-1, 2], [9, -1], [3, 3]])                              # no page, a number beyond the pool, a page
    k.kv4_store(qkv, None, ints([5, 7, -1, 3]), ints([0, 1, 2, 0]), table, pool, heads, kv_heads, d)
    assert torch.equal(pool, before)
    k.kv4_store(qkv[:1], None, ints([64 + 17]), ints([0]), table, pool, heads, kv_heads, d)
    changed = (pool != before).nonzero()[:, 0].unique().tolist()
    assert changed == [2]
    ka, va = k.kv4_load(before, ints([2]), d)
    kb, vb = k.kv4_load(pool, ints([2]), d)
    same = [i for i in range(64) if i != 17]
    eq = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))  # noqa: E731  (random words hold NaN too)
    assert eq(ka[:, :, same], kb[:, :, same]) and eq(va[:, :, same], vb[:, :, same])
    assert torch.equal(kb[0, :, 17].cpu(), rounded4(qkv[0, heads * d:(heads + kv_heads) * d].cpu().view(kv_heads, d)).float().bfloat16())


def test_store_of_values_that_are_not_finite_and_of_equal_ones():
    k = K()
    d = 64
    x = torch.randn(6, 4 * d).bfloat16()
    x[0, 2 * d + 3], x[1, 2 * d + 40], x[2, 3 * d + 1] = math.inf, math.nan, -math.inf
    x[3, 2 * d:3 * d] = 1.25
    x[4, 2 * d:4 * d] = 0.0
    x[5, 2 * d:3 * d] = torch.tensor([3e38, -3e38] * 32).bfloat16()         # a range that float32 does not hold
    pool = k.kv4_pool(1, 1, d, DEV)
    k.kv4_store(x.to(DEV), None, torch.arange(6, dtype=torch.int32, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV), ints([[0]]), pool, 2, 1, d)
    ko, vo = k.kv4_load(pool, ints([0]), d)
    for got, want in ((ko, x[:, 2 * d:3 * d]), (vo, x[:, 3 * d:])):
        got, want = got[0, 0, :6].cpu(), rounded4(want).float().bfloat16()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert bool((ko[0, 0, 3] == 1.25).all()) and bool((ko[0, 0, 4] == 0).all()) and bool(ko[0, 0, 5].isnan().all())
    assert bool(ko[0, 0, 0, :32].isnan().all()) and bool(ko[0, 0, 0, 32:].isfinite().all())


def test_load_gives_zeros_for_numbers_that_are_no_pages():
    k = K()
    pool = torch.randint(0, 100, (3, 2, k.kv4_page_bytes(128)), dtype=torch.uint8, device=DEV)
    ko, vo = k.kv4_load(pool, ints([1, -1, 3, 1]), 128)
    assert bool((ko[1:3] == 0).all()) and bool((vo[1:3] == 0).all()) and torch.equal(ko[0], ko[3])
    assert k.kv4_load(pool, ints([]), 128)[0].shape == (0, 2, 64, 128)


# ---- attention -----------------------------------------------------------------------------------------------------------------

LAYOUTS = [(4, 4, 64), (6, 2, 64), (16, 2, 64), (24, 2, 64), (4, 4, 128), (7, 1, 128), (8, 2, 128), (16, 1, 128)]


@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("window", [0, 40])
def test_single_tokens(heads, kv_heads, d, window):
    c = Case([(n, 1) for n in (0, 1, 15, 16, 31, 32, 63, 64, 65, 127, 128, 200, 333)], heads, kv_heads, d, seed=heads + d)
    c.check(c.run(window, tiles=False), window)


@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("window", [0, 25])
def test_a_few_tokens(heads, kv_heads, d, window):
    c = Case([(0, 3), (62, 4), (130, 2), (5, 1), (64, 5)], heads, kv_heads, d, seed=heads + d + 1)
    c.check(c.run(window, tiles=False), window)


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (16, 2, 64), (6, 2, 128), (8, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("window", [0, 100])
def test_prompts(heads, kv_heads, d, window):
    c = Case([(0, 200), (70, 129), (33, 1), (0, 0), (300, 64)], heads, kv_heads, d, seed=heads + d + 2)
    c.check(c.run(window), window, only=(0, 1, 63, 64, 127, 128, 199))


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (16, 2, 64), (8, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("walks", [True, False])
def test_some_new_tokens_either_way(heads, kv_heads, d, window, walks, monkeypatch):
    """Rows of 1 to 128 new tokens, by the codes and by unpacked pages, whatever the model of both picks."""
    monkeypatch.setattr(K(), "_kv4_walks", lambda *a: walks)
    c = Case([(900, 128), (70, 33), (0, 1), (5, 0), (300, 64), (0, 17)], heads, kv_heads, d, seed=heads + d + 3)
    c.check(c.run(window), window, only=(0, 1, 16, 32, 63, 64, 127))


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128)])
def test_chunks_are_joined(heads, kv_heads, d):
    """A long row in many chunks beside short ones, and the same row alone."""
    from exl3_server_b200.engine.batch import Workspace
    c = Case([(3000, 1), (2, 1), (700, 1)], heads, kv_heads, d, seed=3, q_scale=2.0)
    out = c.run(tiles=False, workspace=Workspace(torch.device(DEV)))
    c.check(out)
    again = c.run(tiles=False, workspace=Workspace(torch.device(DEV)))
    assert torch.equal(out, again)


def test_one_token_prompts_agree_with_single_tokens():
    """row_start None: every row one token."""
    c = Case([(100, 1), (9, 1)], 8, 2, 128, seed=5)
    a = c.run(tiles=False)
    b = K().kv4_attn(c.q, c.pool, c.table, None, c.pos0, None, 1, c.max_len, 8, 2, 128, 128 ** -0.5)
    assert torch.equal(a, b)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_rows_that_see_nothing_get_zeros(d, new):
    c = Case([(40, new), (40, new)], 4, 2, d, seed=6)
    c.table[0] = -1                                                     # a row without any page
    out = c.run().view(2, new, -1)
    assert bool((out[0] == 0).all()) and bool((out[1] != 0).any())
    if new == 1:
        c.pos0[1] = -1                                                  # a row before its first position
        assert bool((c.run() == 0).all())


def test_pages_that_were_given_back_are_left_out():
    c = Case([(400, 1)], 4, 2, 64, seed=7)
    c.table[0, 1:3] = -1
    out = c.run(tiles=False).double().cpu().view(4, 64)
    want = attend(c.q.cpu().view(1, 4, 64), c.k[0], c.v[0], 400, 64 ** -0.5, hidden_keys=set(range(64, 192)))[0]
    assert float((out - want).abs().max()) <= 2.0 ** -7 * float(c.v[0].abs().max())


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 1, 128)])
def test_values_that_a_query_does_not_see_may_be_nan(heads, kv_heads, d):
    """Three new tokens of which the last has NaN keys and values: the first two are as without it, the last is NaN.  (All other
    places of the pages hold NaN words anyway.)"""
    c = Case([(50, 3)], heads, kv_heads, d, seed=8)
    clean = c.run(tiles=False)
    bad = c.qkv[52:53].clone()
    bad[:, heads * d:] = math.nan
    K().kv4_store(bad, None, ints([52]), ints([0]), c.table, c.pool, heads, kv_heads, d)
    out = c.run(tiles=False)
    assert torch.equal(out[:2], clean[:2]) and bool(out[2].isnan().all())


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (8, 1, 128)])
def test_prompts_do_not_see_later_nan(heads, kv_heads, d):
    """The 61st of 150 new tokens has a NaN value: queries before it are as without it, the others NaN."""
    c = Case([(50, 150)], heads, kv_heads, d, seed=15)
    clean = c.run()
    bad = c.qkv[110:111].clone()
    bad[:, (heads + kv_heads) * d + 3] = math.nan                         # the first value head only
    K().kv4_store(bad, None, ints([110]), ints([0]), c.table, c.pool, heads, kv_heads, d)
    out = c.run().view(150, heads, d)
    clean = clean.view(150, heads, d)
    g = heads // kv_heads
    assert torch.equal(out[:60], clean[:60]) and bool(out[60:, :g].isnan().all()) and torch.equal(out[:, g:], clean[:, g:])


def test_a_group_of_values_that_is_nan_stays_in_its_features():
    c = Case([(80, 1)], 4, 4, 64, seed=9)
    bad = c.qkv[10:11].clone()
    bad[:, 4 * 64 + 4 * 64 + 5] = math.inf                                # value head 0, feature 5
    K().kv4_store(bad, None, ints([10]), ints([0]), c.table, c.pool, 4, 4, 64)
    out = c.run(tiles=False).view(4, 64).cpu()
    assert bool(out[0, :32].isnan().all()) and bool(out[0, 32:].isfinite().all()) and bool(out[1:].isfinite().all())
    c.v[0][10, 0, :32] = 0.0
    want = attend(c.q.cpu().view(1, 4, 64), c.k[0], c.v[0], 80, 64 ** -0.5)[0]
    err = (out.double() - want).abs()
    err[0, :32] = 0
    assert float(err.max()) <= 2.0 ** -7 * float(c.v[0].abs().max())


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("new,window", [(1, 0), (2, 30), (90, 0)])
def test_what_lies_in_unused_places_does_not_matter(heads, kv_heads, d, new, window):
    """Places behind the last token, and before the window, hold keys and values of 1e30."""
    c = Case([(100, new)], heads, kv_heads, d, seed=16)
    want = c.run(window)
    n = 100 + new
    width = (heads + 2 * kv_heads) * d
    places = list(range(n, c.table.shape[1] * 64)) + (list(range(0, 100 - 30 + 1 - 1)) if window else [])
    huge = (torch.randn(len(places), width, device=DEV) * 1e30).bfloat16()
    K().kv4_store(huge, None, ints(places), ints([0] * len(places)), c.table, c.pool, heads, kv_heads, d)
    assert torch.equal(c.run(window), want)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("new", [1, 80])
def test_queries_that_are_not_finite(value, new):
    c = Case([(70, new)], 4, 2, 64, seed=10)
    q = c.q.clone()
    q[0, 70] = value                                                    # head 1 of the first token
    out = c.run(q=q).view(new, 4, 64)
    assert bool(out[0, 1].isnan().all()) and bool(out[0, [0, 2, 3]].isfinite().all()) and bool(out[1:].isfinite().all())


@pytest.mark.parametrize("exponent", [-60, -12, 0, 12])
@pytest.mark.parametrize("new", [2, 70])
def test_sizes_of_queries_keys_and_values(exponent, new):
    """Powers of two in q and in k and v move nothing but the result's size (k up, q down: the same scores)."""
    if new == 70 and exponent == -60:
        pytest.skip("fp16 pages hold values down to 2^-24")
    c = Case([(90, new)], 4, 2, 64, seed=11)
    base = c.run()
    f = 2.0 ** exponent
    qkv = c.qkv.clone()
    K().kv4_store((qkv.float() * f).bfloat16(), None, ints(list(range(90 + new))), ints([0] * (90 + new)), c.table, c.pool, 4, 2, 64)
    out = c.run(q=(c.q.float() / f).bfloat16())
    tol = 2.0 ** -7 if exponent >= 0 or new == 2 else 2.0 ** -5              # (fp16 has fewer bits below 2^-14)
    assert float((out.double() / f - base.double()).abs().max()) <= tol * float(c.v[0].abs().max())


def test_places_beyond_32_bits():
    """A pool of more than 4 GiB whose last pages are used."""
    k = K()
    d, g = 128, 8
    pages = (5 << 30) // (g * k.kv4_page_bytes(d))
    pool = torch.empty((pages, g, k.kv4_page_bytes(d)), dtype=torch.uint8, device=DEV)
    n = 150
    table = torch.arange(pages - 3, pages, dtype=torch.int32, device=DEV)[None]
    x = torch.randn(n, (16 + 2 * g) * d, generator=torch.Generator().manual_seed(12)).bfloat16()
    q = k.kv4_store(x.to(DEV), None, torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV), table, pool, 16, g, d)
    kk, vv = (rounded4(x[:, o * d:(o + g) * d].view(n, g, d)) for o in (16, 16 + g))
    for new in (1, n):
        tiles = (ints([0] * (-(-new // 128))), ints(list(range(0, new, 128))), -(-new // 128))
        out = k.kv4_attn(q[n - new:], pool, table, ints([0, new]), ints([n - new]), tiles, new, n, 16, g, d, d ** -0.5)
        want = attend(x[n - 1:, :16 * d].view(1, 16, d), kk, vv, n - 1, d ** -0.5)[0]
        assert float((out[-1].double().cpu().view(16, d) - want).abs().max()) <= 2.0 ** -6 * float(vv.abs().max())


def test_on_another_stream_and_in_a_graph():
    c = Case([(700, 1), (64, 1)], 8, 2, 128, seed=13)
    want = c.run(tiles=False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run(tiles=False)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    from exl3_server_b200.engine.batch import Workspace
    ws, out = Workspace(torch.device(DEV), keep_outgrown=True), torch.empty_like(want)
    c.run(tiles=False, workspace=ws, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(tiles=False, workspace=ws, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    K().check_status()


def test_refusals():
    from exl3_server_b200.ops.lib import KernelLibraryError as E
    k = K()
    c = Case([(10, 1)], 4, 2, 64, seed=14)
    one = ints([0])
    for f in (
        lambda: k.kv4_page_bytes(96),
        lambda: k.kv4_pool(1, 1, 80, DEV),
        lambda: k.kv4_store(c.qkv.float(), None, one, one, c.table, c.pool, 4, 2, 64),
        lambda: k.kv4_store(c.qkv, None, one, one, c.table, c.pool, 3, 2, 64),
        lambda: k.kv4_store(c.qkv, None, one, one, c.table, c.pool, 4, 2, 64),                       # one position for eleven tokens
        lambda: k.kv4_store(c.qkv[:1], torch.zeros(16, device=DEV), one, one, c.table, c.pool, 4, 2, 64),
        lambda: k.kv4_store(c.qkv[:1], None, one.long(), one, c.table, c.pool, 4, 2, 64),
        lambda: k.kv4_store(c.qkv[:1].cpu(), None, one, one, c.table, c.pool, 4, 2, 64),
        lambda: k.kv4_load(c.pool.float(), one, 64),
        lambda: k.kv4_load(c.pool, one, 128),
        lambda: c.run(q=c.q.float()),
        lambda: k.kv4_attn(c.q, c.pool, c.table, c.start, c.pos0, None, 1, 11, 4, 3, 64, 0.125),
        lambda: k.kv4_attn(c.q, c.pool, c.table, ints([0]), c.pos0, None, 1, 11, 4, 2, 64, 0.125),
        lambda: k.kv4_attn(c.q, c.pool, c.table, None, c.pos0, None, 2, 11, 4, 2, 64, 0.125),
        lambda: k.kv4_attn(c.q, c.pool, c.table, c.start, c.pos0, None, 1, 11, 4, 2, 64, 0.125, window=-1),
        lambda: k.kv4_attn(c.q, c.pool, c.table, c.start, c.pos0, None, 1, 11, 4, 2, 64, 0.125, out=c.q[:, :64]),
    ):
        with pytest.raises(E):
            f()
