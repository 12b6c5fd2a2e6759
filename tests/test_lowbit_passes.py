"""How the prompt form of the 4-bit cache's attention divides a step's rows into passes over its scratch memory (host side)."""
import random

import pytest

from exl3_server_b200.engine.batch import Workspace, pack_step
from exl3_server_b200.ops import kernels as K


def plan(row_pages, total, page_bytes):
    return K._kv4_passes(1, 1, row_pages, total, 1, 1, 1, page_bytes // 256, K.KV4_PROMPT_BYTES)[:3]


@pytest.mark.parametrize("seed", range(40))
def test_every_pass_holds_its_rows(seed):
    rng = random.Random(seed)
    page_bytes = 4 * 64 * rng.choice([64, 128]) * rng.choice([1, 8, 36])
    pages = [rng.choice([0, 1, 4, rng.randint(1, 600)]) for _ in range(rng.randint(1, 200))]
    row_pages, total = max(1, max(pages)), max(1, sum(pages))
    slots, stride, passes = plan(row_pages, total, page_bytes)
    used, before = {}, 0
    for n in pages:
        p = min(before // stride, passes - 1)
        if n:
            assert before // stride == p
        used[p] = used.get(p, 0) + n
        before += n
    assert all(0 <= p < passes for p in used) and max(used.values()) <= slots
    assert slots <= max(total if passes == 1 else 0, 2 * row_pages, K.KV4_PROMPT_BYTES // page_bytes)
    if total * page_bytes <= K.KV4_PROMPT_BYTES:
        assert passes == 1


def test_scratch_of_one_long_prompt_among_short_ones():
    """36 heads of 64 with keys of their own: 32,768 tokens and 63 times 200."""
    lens = [(0, 32768)] + [(0, 200)] * 63
    sizes = [K._kv4_row_pages(c, n, 0, 512) for c, n in lens]
    page_bytes = 4 * 36 * 64 * 64
    slots, _, passes = plan(max(sizes), sum(sizes), page_bytes)
    assert passes == 1 and slots == 512 + 63 * 4 and slots * page_bytes < 0.46e9
    many = [512] * 64
    slots, _, passes = plan(512, sum(many), page_bytes)
    assert passes > 1 and slots * page_bytes <= max(K.KV4_PROMPT_BYTES, 2 * 512 * page_bytes)


@pytest.mark.parametrize("ctx,new,window,width,want", [
    (0, 1, 0, 9, 1), (0, 64, 0, 9, 1), (0, 65, 0, 9, 2), (63, 1, 0, 9, 1), (64, 1, 0, 9, 2), (1000, 0, 0, 99, 0), (1000, 24, 0, 3, 3),
    (1000, 24, 100, 99, 2), (1000, 24, 1, 99, 1), (1000, 25, 1, 99, 2), (1000, 24, 100, 10, 0), (128, 2, 66, 99, 3 - 0), (128, 2, 65, 99, 2),
])
def test_pages_that_a_row_sees(ctx, new, window, width, want):
    assert K._kv4_row_pages(ctx, new, window, width) == want
    seen = {p // 64 for q in range(ctx, ctx + new) for p in range(max(0, q - window + 1) if window else 0, q + 1) if p // 64 < width}
    assert want == len(seen)


def test_a_step_carries_its_rows_lengths():
    b = pack_step([0, 1], [5, 0], [[1, 2], [3]], [[], []], [[[0], [1]]], Workspace("cpu"), "cpu")
    assert b.row_lens == ((5, 2), (0, 1))


def test_which_rows_walk_beside_prompts():
    """Rows of up to 4 tokens walk where they have enough keys together, and then up to the longest of them; the others' pages are counted."""
    lens = ((8000, 1), (7000, 2), (0, 200), (100, 5), (5, 0))
    assert K._kv4_rows(lens, 4, 15003, 0, 999) == (2, 8001, 4, 4 + 2)
    assert K._kv4_rows(lens, 4, 15004, 0, 999) == (0, 0, 126, 126 + 110 + 4 + 2)
    assert K._kv4_rows(lens, 4, 203, 100, 999) == (2, 8001, 4, 4 + 2)
    assert K._kv4_rows(lens, 4, 204, 100, 999)[0] == 0
    assert K._kv4_rows(((0, 200), (3, 0)), 4, 0, 0, 999) == (0, 0, 4, 4)
