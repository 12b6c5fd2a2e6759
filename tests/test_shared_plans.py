"""What a call of attention over shared pages settles before anything is launched: its scratch memory against what its kernels write into it, worked out here.  On the CPU."""
import random
import weakref

import pytest
import torch

from exl3_server_b200.ops import kernels as K

SMS = 148


def tiles_made(news, groups, heads_per, many):
    """Tiles of a key/value head that a step's kernel makes: of each group's queries, and of each row's own where rows of many tokens have tiles."""
    first = 0
    tiles = 0
    for n in groups:
        tiles += -(-sum(news[first:first + n]) * heads_per // 256)
        first += n
    return tiles + (sum(-(-n * heads_per // 256) for n in news if n * heads_per > 64) if many else 0)


def floats_written(tiles, T, heads, kv_heads, d):
    """The counters, the walk's records, the tiles' places and parts, the tokens' and the rows' own parts, each at least as far as it is written."""
    walk = SMS * (8 * 16 * d + 2 * 16 * (d + 2))
    return 65536 + walk + 4 * kv_heads * tiles + 4 * T + (SMS - 1 + kv_heads * tiles) * 256 * (d + 2) + T * heads * (d + 2)


def check(news, groups, heads, kv_heads, d, width):
    T = sum(news)
    need, used, many, most = K._shared_plan(SMS, T, len(news), heads, kv_heads, d, len(groups), max(news), width)
    assert used in (0, len(groups))
    tiles = tiles_made(news, groups if used else [], heads // kv_heads, many)
    assert tiles <= most <= 512
    if most:
        assert need >= floats_written(tiles, T, heads, kv_heads, d), (need, used, many, most)
    return used, many, most


@pytest.mark.parametrize("rows,new,heads,kv_heads,groups,width", [
    (300, 5, 16, 1, 32, 1), (300, 5, 16, 1, 32, 4), (300, 10, 8, 1, 30, 2), (300, 16, 20, 4, 32, 1), (300, 16, 20, 4, 100, 1)])
def test_groups_that_are_left_alone(rows, new, heads, kv_heads, groups, width):
    """Without its groups such a call gives each row a tile of its own, and with them not: its scratch memory has to be that of the tiles it has."""
    cuts = [rows * i // groups for i in range(groups + 1)]
    used, many, most = check([new] * rows, [b - a for a, b in zip(cuts, cuts[1:])], heads, kv_heads, 64, width)
    assert used == 0 and many and most >= rows


@pytest.mark.parametrize("news,heads,kv_heads,d,groups,width,want", [
    ([98] * 62, 32, 1, 128, [20, 20, 22], 18, (0, False)),              # 759 tiles and more of the groups alone
    ([8192], 32, 2, 128, [1], 400, (0, False)),                         # 512 and one
    ([5, 8180], 32, 2, 128, [1], 400, (1, False)),                      # 512
    ([1] * 512, 128, 1, 128, [2] * 256, 300, (256, False)),             # 512
    ([1] * 514, 128, 1, 128, [2] * 256, 300, (0, False)),               # 513
    ([1] * 64, 32, 8, 128, [64], 1 << 19, (1, False)),
    ([1] * 64, 16384, 4096, 128, [64], 1 << 19, (0, False)),            # 2 tiles of 4,096 heads and 2^19 pages: more than 31 bits hold
])
def test_groups_are_never_why_a_call_is_refused(news, heads, kv_heads, d, groups, width, want):
    """They say what may be read once: where their tiles are too many, rows read for themselves."""
    assert check(news, groups, heads, kv_heads, d, width)[:2] == want


@pytest.mark.parametrize("news,heads,kv_heads,groups,want", [
    ([8191], 64, 8, [], (True, 256)), ([8192], 64, 8, [], (True, 257)), ([4096], 32, 2, [], (True, 257)), ([8150], 32, 2, [], (True, 510)),
    ([8176], 32, 2, [], (True, 512)), ([8192], 32, 2, [], (False, 0)),
    ([100] * 60, 32, 2, [], (True, 435)), ([100] * 60, 32, 2, [60], (False, 376)),             # (a group's tiles are counted beside the rows')
])
def test_prompts_have_tiles_up_to_what_the_list_holds(news, heads, kv_heads, groups, want):
    assert check(news, groups, heads, kv_heads, 64, 300)[1:] == want


@pytest.mark.parametrize("seed", range(8))
def test_scratch_holds_what_is_written(seed):
    """Rows, groups and tables on both sides of the limits."""
    rng = random.Random(seed)
    seen = set()
    for _ in range(1500):
        heads, kv_heads, d = rng.choice([(16, 2, 64), (16, 1, 64), (8, 1, 64), (20, 4, 64), (36, 36, 64), (32, 8, 128), (32, 1, 128), (7, 1, 128), (128, 1, 128)])
        rows = int(2 ** rng.uniform(0, 10.2))
        high = int(2 ** rng.uniform(0, min(13, 17.5 - rng.uniform(0, 1) * rows.bit_length())))
        news = [rng.randint(0, max(high, 1)) for _ in range(rows)]
        news[rng.randrange(rows)] = max(high, 1)
        left, groups = rows, []
        while left and len(groups) < 256 and rng.random() < 0.97:
            groups.append(min(left, rng.choice([1, 2, 3, 10, 40])))
            left -= groups[-1]
        seen.add(check(news, groups, heads, kv_heads, d, int(2 ** rng.uniform(0, 9)))[:2])
    assert len({many for _, many in seen}) == 2


@pytest.mark.parametrize("lists", [False, True])
def test_scratch_memory_lives_until_the_launch(lists, monkeypatch):
    """Without a workspace: memory that is free when the kernels go into the stream may be another thread's by then."""
    made, alive = [], []
    zeros = torch.zeros

    def note(*a, **kw):
        t = zeros(*a, **kw)
        made.append(weakref.ref(t))
        return t

    def entry(name, args):
        def call(*values):
            alive.append([r() is not None and r().data_ptr() in values for r in made])
            return 0
        return call

    q, pool, table = zeros(3, 256).bfloat16(), zeros(4, 2, 64, 64).bfloat16(), zeros(2, 2, dtype=torch.int32)
    row_start, pos0, pos, seq, pages = (torch.tensor(v, dtype=torch.int32) for v in ([0, 1, 3], [5, 70], [5, 70, 71], [0, 1, 1], [[[0], [0]]] * 3))
    monkeypatch.setattr(K, "_entry", entry)
    monkeypatch.setattr(K, "_on_this_device", lambda *a: None)
    monkeypatch.setattr(K, "_raw_stream", lambda: 0)
    monkeypatch.setattr(K, "_sms", lambda t: SMS)
    monkeypatch.setattr(K.torch, "zeros", note)
    if lists:
        K.attn_pages(q, pool, pool, table, pos, seq, pages, 4, 2, 64, scale=0.1)
    else:
        K.attn_shared(q, pool, pool, table, row_start, pos0, None, 2, 4, 2, 64, scale=0.1)
    assert alive == [[True]]


@pytest.mark.parametrize("rows,heads,groups,width", [(4, 8, 1, 20), (30, 2, 0, 20), (64, 8, 1, 200), (1500, 8, 3, 200)])
def test_no_row_brings_more_than_all_tokens(rows, heads, groups, width):
    """``max_new`` is a bound: one far above the tokens that there are changes nothing."""
    plans = {K._shared_plan(SMS, rows, rows, heads, 1, 64, groups, most, width) for most in (rows, 1 << 24, 2 ** 31 - 1)}
    assert len(plans) == 1


@pytest.mark.parametrize("off", [1, 4])
def test_codes_of_bounds_that_are_not_aligned(off):
    """Refused by all that read or write them, before anything is launched."""
    flat = torch.zeros(4 * 2 * 2 * 64 + 16, dtype=torch.int8)
    codes = flat[(-flat.data_ptr()) % 16 + off:].data_ptr()
    x = torch.zeros(4096, dtype=torch.float32)
    p = x.data_ptr() + (-x.data_ptr()) % 16
    for call in (
        lambda: K._entry("exl3_page_bounds_load", "pplpiiipp")(codes, p, 4, p, 1, 2, 64, p, p, 0),
        lambda: K._entry("exl3_page_bounds", "plpiippiiiipp")(p, 4, p, 2, 2, p, p, 1, 1, 2, 64, codes, p, 0),
        lambda: K._entry("exl3_page_select", "plpplpiiippiiiiiiip")(p, 256, codes, p, 4, p, 2, 2, 1, p, p, 1, 4, 2, 64, 1, 1, 1, p, 0),
    ):
        with pytest.raises(K.KernelLibraryError, match="aligned"):
            K._check(call(), "bounds")
