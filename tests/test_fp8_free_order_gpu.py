"""Products of up to 8 rows in 8-bit floating point that may be added up in any order (``fixed_order=False``), against plain float64.

Tolerances, fixed before the first run, are test_fp8_gpu.py's: with S = sum |x| |w| of the rounded values float32 sums are off by at most 2^-17 S; a
bfloat16 result adds 2^-9 of itself; silu(gate) * up as there."""
import math

import pytest
import torch

from plain_lowbit import product8
from test_fp8_gpu import DEV, F, K, make, sizes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize("N,Kd", [(1, 16), (16, 128), (200, 272), (333, 1040), (2304, 144), (2500, 2304), (5000, 1024), (130, 8192), (40, 8208), (128, 6656)])
def test_product(M, N, Kd):
    x, w, s = make(M, N, Kd, seed=M + N)
    bias = torch.randn(N, device=DEV).bfloat16() if (M + N) % 2 else None
    want, size = product8(x, w, s, bias), sizes(x, w, s)
    for out_dtype, own in ((torch.float32, 2.0 ** -22), (torch.bfloat16, 2.0 ** -8)):
        y = K().fp8_linear(x, w, s, bias=bias, out_dtype=out_dtype, fixed_order=False)
        assert y.dtype == out_dtype and y.shape == (M, N)
        bound = 2.0 ** -17 * size + own * want.abs() + 1e-30
        assert bool(((y.to(F) - want).abs() <= bound).all()), float(((y.to(F) - want).abs() / bound).max())
        assert torch.equal(y, K().fp8_linear(x, w, s, bias=bias, out_dtype=out_dtype, fixed_order=False))
    K().check_status()


@pytest.mark.parametrize("M", [1, 4, 8])
@pytest.mark.parametrize("N,Kd", [(16, 128), (272, 272), (4096, 1040), (6144, 2304)])
def test_gated_product(M, N, Kd):
    x, w, s = make(M, N, Kd, seed=M + N + 1, x_scale=0.5)
    want = product8(x, w, s, gated=True)
    z, size = product8(x, w, s).view(M, N // 16, 2, 8), sizes(x, w, s).view(M, N // 16, 2, 8)
    gate, up = z[:, :, 0], z[:, :, 1]
    for out_dtype, own in ((torch.float32, 2.0 ** -18), (torch.bfloat16, 2.0 ** -8)):
        y = K().fp8_linear(x, w, s, out_dtype=out_dtype, gated=True, fixed_order=False)
        bound = (2.0 ** -17 * (1.1 * size[:, :, 0] * up.abs() + gate.abs() * size[:, :, 1])).reshape(M, N // 2) + own * want.abs() + 1e-7
        assert y.shape == (M, N // 2) and bool(((y.to(F) - want).abs() <= bound).all())


def test_rows_that_are_not_finite_stay_by_themselves():
    x, w, s = make(5, 300, 400, seed=4)
    clean = K().fp8_linear(x, w, s, fixed_order=False)
    x[1, 7], x[3, 399] = math.nan, -math.inf
    y = K().fp8_linear(x, w, s, fixed_order=False)
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().all())
    assert torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


def test_rows_apart_and_another_stream():
    x, w, s = make(4, 384, 512, seed=5)
    wide = torch.full((4, 600), math.nan, device=DEV).bfloat16()
    wide[:, 40:552] = x
    want = K().fp8_linear(x, w, s, fixed_order=False)
    out = torch.zeros(4, 384, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K().fp8_linear(wide[:, 40:552], w, s, out=out, fixed_order=False)
    torch.cuda.current_stream().wait_stream(side)
    assert got is out and torch.equal(out, want)


@pytest.mark.parametrize("M,N,Kd", [(1, 2304, 2304), (4, 6144, 4096), (8, 1024, 1024)])
def test_products_in_a_chain(M, N, Kd):
    """Launches that overlap: each may begin before the one that wrote its input has ended."""
    x, w, s = make(M, N, Kd, seed=6)
    back, bs = K().fp8_quantize_weight(torch.randn(Kd, N, device=DEV).bfloat16() * (0.5 / N ** 0.5))
    def run():
        y = x
        for _ in range(6):
            y = K().fp8_linear(K().fp8_linear(y, w, s, fixed_order=False), back, bs, fixed_order=False)
        return y
    first = run()
    torch.cuda.synchronize()
    y = x
    for _ in range(6):
        z = K().fp8_linear(y, w, s, fixed_order=False)
        torch.cuda.synchronize()
        y = K().fp8_linear(z, back, bs, fixed_order=False)
        torch.cuda.synchronize()
    assert bool(y.isfinite().all()) and torch.equal(first, y)
    assert all(torch.equal(run(), first) for _ in range(20))


def test_refusals():
    from exl3_server_b200.ops.lib import KernelLibraryError
    x, w, s = make(2, 64, 128, seed=7)
    wide = torch.zeros(128, device=DEV).bfloat16()
    for kw in (dict(bias=wide[::2]), dict(bias=wide), dict(bias=wide[:64].float()), dict(bias=wide[:64], gated=True)):
        with pytest.raises(KernelLibraryError, match="bias"):
            K().fp8_linear(x, w, s, fixed_order=False, **kw)
    with pytest.raises(KernelLibraryError):
        K().fp8_linear(x.cpu(), w, s, fixed_order=False)
    assert K().fp8_linear(x[:0], w, s, fixed_order=False).shape == (0, 64)
