"""What needs no GPU of the 8-bit weights and the 4-bit cache: refusals before anything is read, the cache's sizes, the chunks of the
attention's rows, the weights' rounding on the host."""
import math

import pytest
import torch

from exl3_server_b200 import LlamaConfig, load_model, write_random_model
from exl3_server_b200.cache.kv import SequenceCache
from exl3_server_b200.cache.pages import CacheError
from exl3_server_b200.cli import build_parser
from exl3_server_b200.ops import kernels as K
from exl3_server_b200.ops.lib import KernelLibraryError
from exl3_server_b200.parts.base import KVRequest
from plain_lowbit import e4m3, page_values, rounded4


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    cfg = LlamaConfig(hidden_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1, head_dim=32, intermediate_size=96, vocab_size=64)
    return write_random_model(cfg, str(tmp_path_factory.mktemp("m") / "a"), seed=1)


@pytest.mark.parametrize("kw,said", [
    (dict(dtype="float32", weight_type="fp8"), "bfloat16"), (dict(dtype="float32", cache_type="int4"), "bfloat16"),
    (dict(weight_type="int3"), "weight_type"), (dict(cache_type="fp8"), "cache_type"), (dict(cache_type="int4"), "heads of 64 or 128"),
])
def test_types_that_are_refused(folder, kw, said):
    with pytest.raises(ValueError, match=said):
        load_model(folder, device="cpu", **kw)


def test_other_decoders_are_refused(tmp_path):
    from nibelix_configs import CONFIGS, make_nibelix
    d = make_nibelix(sorted(CONFIGS)[0], str(tmp_path / "n"))
    for kw in (dict(weight_type="fp8"), dict(cache_type="int4")):
        with pytest.raises(ValueError, match="does not keep"):
            load_model(d, device="cpu", **kw)


def test_input_features_that_are_refused(tmp_path):
    cfg = LlamaConfig(hidden_size=72, num_hidden_layers=1, num_attention_heads=1, num_key_value_heads=1, head_dim=64, intermediate_size=96, vocab_size=64)
    d = write_random_model(cfg, str(tmp_path / "b"), seed=1)
    with pytest.raises(ValueError, match="multiples of 16"):
        load_model(d, device="cpu", weight_type="fp8")


def test_flags():
    a = build_parser().parse_args(["--model", "x", "--weight-type", "fp8", "--cache-type", "int4"])
    assert (a.weight_type, a.cache_type) == ("fp8", "int4")
    b = build_parser().parse_args(["--model", "x"])
    assert b.weight_type is None and b.cache_type is None


def test_cache_sizes_and_guards():
    full, four = KVRequest(2, 64), KVRequest(2, 64, codes=4)
    c = SequenceCache([(full, None, None), (four, None, None), (four, None, None)], 256, device="cpu")
    assert len(c.groups) == 2
    g = c.groups[1]
    assert g.k is g.v and g.k.dtype == torch.uint8 and tuple(g.k.shape) == (2, 5, 2, K.kv4_page_bytes(64))
    assert g.bytes_per_token(2) == 2 * 2 * 80 and c.groups[0].bytes_per_token(2) == 2 * 128 * 2
    assert g.guards_intact() and g.k.data_ptr() % 16 == 0
    g._k_store[-1] = 0
    assert not g.guards_intact()
    with pytest.raises(CacheError):
        c.check_guards()
    with pytest.raises(CacheError, match="pages of 64"):
        SequenceCache([(four, None, None)], 256, device="cpu", page_size=32)
    with pytest.raises(CacheError, match="head shapes"):
        SequenceCache([(full, None, None), (four, None, 0)], 256, device="cpu")


def test_page_bytes():
    assert (K.kv4_page_bytes(64), K.kv4_page_bytes(128)) == (5120, 10240)
    for d in (0, 32, 96, 256):
        with pytest.raises(KernelLibraryError):
            K.kv4_page_bytes(d)


@pytest.mark.parametrize("rows", [1, 5, 64])
@pytest.mark.parametrize("span", [1, 31, 64, 65, 1000, 131072, 1000000])
@pytest.mark.parametrize("columns,head_dim,window", [(4, 64, 0), (8, 128, 0), (16, 128, 512)])
def test_chunks_cover_every_row(rows, span, columns, head_dim, window):
    chunk, n = K._kv4_chunks(rows, 2, 3, columns, head_dim, span, window, 148)
    per = 4096 // head_dim
    assert 1 <= chunk <= 128 and n >= 1
    if not window:
        assert chunk * n >= -(-span // per)
    else:                                                   # from wherever the window begins to its end
        assert n >= max((at + span - 1) // per // chunk - at // per // chunk + 1 for at in range(0, chunk * per, 7))


def test_weights_rounding_on_the_host():
    w = torch.randn(200, 300, generator=torch.Generator().manual_seed(1)) * 0.1
    codes, scales = K.fp8_quantize_weight(w)
    assert codes.dtype == torch.float8_e4m3fn and tuple(scales.shape) == (2, 3)
    back = codes.float() * scales.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300]
    assert float((back - w).abs().max()) <= 2.0 ** -4 * float(w.abs().max())
    assert math.isclose(float(codes.float().abs().max()), 448.0)


def test_the_plain_forms_agree_with_torch():
    x = torch.randn(4000, generator=torch.Generator().manual_seed(2)) * 50
    assert torch.equal(e4m3(x), x.to(torch.float8_e4m3fn).double())
    y = torch.randn(3, 64, generator=torch.Generator().manual_seed(3))
    r = rounded4(y)
    assert float((r - y).abs().max()) <= 0.51 / 15 * float((y.amax() - y.amin())) + 2.0 ** -8 * float(y.abs().max())
    k, v = page_values(torch.zeros(5120, dtype=torch.uint8), 64)
    assert bool((k == 0).all()) and k.shape == (64, 64) and v.shape == (64, 64)


def test_which_way_the_4_bit_attention_goes():
    walks = K._kv4_walks
    # rows, query tiles, heads, key/value heads, head size, new tokens, longest row, visible keys: measured on both sides, far from the edge
    assert walks(1, 1, 32, 2, 128, 5, 30005, 30005) and walks(1, 1, 16, 2, 64, 100, 30100, 30100) and walks(16, 16, 32, 8, 128, 12, 4012, 4012)
    assert not walks(16, 16, 32, 8, 128, 64, 4064, 4064) and not walks(1, 31, 32, 8, 128, 3900, 5100, 5100)
    assert not walks(16, 16, 16, 2, 64, 100, 4100, 4100)
    assert not walks(1, 1, 128 * 65536 // 64, 65536 // 4, 64, 128, 128, 128)              # more groups of columns than a grid has room for
