"""What planning a call of the 4-bit cache's attention costs the host (the plan itself: test_lowbit.py)."""
import pytest

from exl3_server_b200.ops import kernels as K
from exl3_server_b200.ops.lib import KernelLibraryError


@pytest.mark.parametrize("head_dim,first", [(128, 30000), (64, 131072), (128, 1)])
@pytest.mark.parametrize("window", [0, 100000])
def test_a_growing_length_is_planned_once_a_tile(head_dim, first, window):
    """A sequence that grows by a token a step: a plan for each new tile of 4096 / head_dim keys, not for each length."""
    K._kv4_tile_chunks.cache_clear()
    for span in range(first, first + 256):
        K._kv4_chunks(1, 8, 1, 4, head_dim, span, window, 148)
    assert K._kv4_tile_chunks.cache_info().misses <= 256 // (4096 // head_dim) + 1


@pytest.mark.parametrize("span", [30000, 131071, 1000000])
def test_a_plan_tries_each_number_of_chunks_once(span, monkeypatch):
    tried = []
    ceil = K.math.ceil
    monkeypatch.setattr(K.math, "ceil", lambda x: tried.append(x) or ceil(x))       # (one call a candidate)
    K._kv4_tile_chunks.__wrapped__(8, True, 4, 128, -(-span // 32), False, 148)
    assert 0 < len(tried) <= 128


def test_rows_that_are_too_long_are_refused():
    with pytest.raises(KernelLibraryError, match="longer than"):
        K._kv4_chunks(1, 8, 1, 4, 128, 32 * 1024 * 128 + 1, 0, 148)
    assert K._kv4_chunks(1, 8, 1, 4, 128, 32 * 1024 * 128, 0, 148) == (128, 1024)
