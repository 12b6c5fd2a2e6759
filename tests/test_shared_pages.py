"""What the entry points of attention over shared and over chosen pages refuse, before anything is launched: on the CPU."""
import pytest
import torch

from exl3_server_b200.ops import kernels as K
from exl3_server_b200.ops.lib import KernelLibraryError


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def shared_args(**kw):
    a = dict(q=torch.zeros(3, 256).bfloat16(), k_pool=torch.zeros(4, 2, 64, 64).bfloat16(), v_pool=torch.zeros(4, 2, 64, 64).bfloat16(),
             block_table=torch.zeros(2, 2, dtype=torch.int32), row_start=ints(0, 1, 3), row_pos0=ints(5, 70), groups=torch.zeros(1, 3, dtype=torch.int32), max_new=2,
             heads=4, kv_heads=2, head_dim=64, scale=0.125)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(3, 256)), "q must be bfloat16"),
    (dict(q=torch.zeros(3, 255).bfloat16()), "q must be bfloat16"),
    (dict(q=torch.zeros(3, 512).bfloat16()[:, ::2]), "q must be bfloat16"),
    (dict(heads=5), "groups of one size"),
    (dict(head_dim=96), "heads of 64 or 128"),
    (dict(kv_heads=0), "groups of one size"),
    (dict(k_pool=torch.zeros(4, 2, 32, 64).bfloat16()), "k_pool must be"),
    (dict(v_pool=torch.zeros(4, 2, 64, 64)), "v_pool must be"),
    (dict(v_pool=torch.zeros(5, 2, 64, 64).bfloat16()), "different numbers of pages"),
    (dict(k_pool=torch.zeros(4, 64, 2, 64).bfloat16().transpose(1, 2)), "k_pool must be contiguous"),
    (dict(row_start=ints(0, 1)), "row_start has 2 entries for 2 rows"),
    (dict(row_pos0=torch.zeros(2, dtype=torch.int64)), "row_pos0 must be int32"),
    (dict(block_table=torch.zeros(1, 2, dtype=torch.int32)), "block table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), "block table"),
    (dict(groups=torch.zeros(3, dtype=torch.int32)), "groups must be"),
    (dict(groups=torch.zeros(1, 3, dtype=torch.int64)), "groups must be int32"),
    (dict(groups=torch.zeros(257, 3, dtype=torch.int32)), "groups must be"),
    (dict(out=torch.zeros(3, 256)), "out must be"),
    (dict(out=torch.zeros(2, 256).bfloat16()), "out must be"),
    (dict(), "not on a CUDA device"),
])
def test_attn_shared_refuses(change, words):
    with pytest.raises(KernelLibraryError, match=words):
        K.attn_shared(**shared_args(**change))


def pages_args(**kw):
    a = dict(q=torch.zeros(3, 256).bfloat16(), k_pool=torch.zeros(4, 2, 64, 64).bfloat16(), v_pool=torch.zeros(4, 2, 64, 64).bfloat16(),
             block_table=torch.zeros(2, 2, dtype=torch.int32), tok_pos=ints(1, 2, 3), tok_seq=ints(0, 0, 1), pages=torch.zeros(3, 2, 5, dtype=torch.int32), heads=4,
             kv_heads=2, head_dim=64, scale=0.125)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(3, 256)), "q must be bfloat16"),
    (dict(tok_pos=ints(1, 2)), "tok_pos has 2"),
    (dict(tok_seq=torch.zeros(3, dtype=torch.int64)), "tok_seq must be int32"),
    (dict(pages=torch.zeros(3, 5, dtype=torch.int32)), "pages must be int32"),
    (dict(pages=torch.zeros(3, 1, 5, dtype=torch.int32)), "pages must be int32"),
    (dict(pages=torch.zeros(3, 2, 0, dtype=torch.int32)), "pages must be int32"),
    (dict(pages=torch.zeros(3, 2, 5)), "pages must be int32"),
    (dict(pages=torch.zeros(3, 2, 10, dtype=torch.int32)[..., ::2]), "pages must be contiguous"),
    (dict(v_pool=torch.zeros(4, 1, 64, 64).bfloat16()), "v_pool must be"),
    (dict(), "not on a CUDA device"),
])
def test_attn_pages_refuses(change, words):
    with pytest.raises(KernelLibraryError, match=words):
        K.attn_pages(**pages_args(**change))


def select_args(**kw):
    a = dict(q=torch.zeros(3, 256).bfloat16(), codes=torch.zeros(4, 2, 2, 64, dtype=torch.int8), scales=torch.zeros(4, 2), block_table=torch.zeros(2, 2, dtype=torch.int32),
             tok_pos=ints(1, 2, 3), tok_seq=ints(0, 0, 1), count=4, heads=4, kv_heads=2, head_dim=64)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(3, 128).bfloat16()), "q must be bfloat16"),
    (dict(codes=torch.zeros(4, 2, 2, 64)), "codes must be"),
    (dict(codes=torch.zeros(4, 2, 2, 32, dtype=torch.int8)), "codes must be"),
    (dict(scales=torch.zeros(4, 3)), "scales must be"),
    (dict(scales=torch.zeros(4, 2, dtype=torch.float64)), "scales must be"),
    (dict(kv_heads=1), "key/value heads"),
    (dict(tok_pos=ints(1)), "tok_pos has 1"),
    (dict(out=torch.zeros(3, 2, 5, dtype=torch.int32)), "out must be"),
    (dict(count=0), "count of 1 or more"),
    (dict(first=-1), "first -1"),
    (dict(last=0), "last 0"),
    (dict(), "not on a CUDA device"),
])
def test_page_select_refuses(change, words):
    with pytest.raises(KernelLibraryError, match=words):
        K.page_select(**select_args(**change))


def bounds_args(**kw):
    a = dict(k_pool=torch.zeros(4, 2, 64, 64).bfloat16(), codes=torch.zeros(4, 2, 2, 64, dtype=torch.int8), scales=torch.zeros(4, 2),
             block_table=torch.zeros(2, 2, dtype=torch.int32), row_start=ints(0, 1, 3), row_pos0=ints(5, 70), max_new=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(k_pool=torch.zeros(4, 2, 64, 128).bfloat16()), "k_pool must be"),
    (dict(k_pool=torch.zeros(5, 2, 64, 64).bfloat16()), "5 pages of keys, bounds of 4"),
    (dict(codes=torch.zeros(4, 2, 1, 64, dtype=torch.int8)), "codes must be"),
    (dict(row_start=ints(0, 3)), "row_start has 2"),
    (dict(max_new=-1), "max_new -1"),
    (dict(), "not on a CUDA device"),
])
def test_page_bounds_refuses(change, words):
    with pytest.raises(KernelLibraryError, match=words):
        K.page_bounds(**bounds_args(**change))


def test_page_bounds_load_refuses():
    codes, scales = K.page_bounds_pool(4, 2, 64, "cpu")
    for pages, words in ((ints(0).long(), "int32"), (ints(0), "not on a CUDA device")):
        with pytest.raises(KernelLibraryError, match=words):
            K.page_bounds_load(codes, scales, pages)
    with pytest.raises(KernelLibraryError, match="64 or 128"):
        K.page_bounds_pool(4, 2, 96, "cpu")


def test_scales_that_are_refused():
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(KernelLibraryError, match="positive"):
            K.attn_shared(**shared_args(scale=scale))
        with pytest.raises(KernelLibraryError, match="positive"):
            K.attn_pages(**pages_args(scale=scale))
