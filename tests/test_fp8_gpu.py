"""Products in 8-bit floating point with scales for blocks of 128, against plain float64; refusals.

Tolerances, fixed before the first run: codes and scales are exact.  A product's sums are float32 over codes that are exact: with S = sum |x| |w| (of
the rounded values) they are off by at most K / 128 + 16 roundings of 2^-24 S, 2^-17 S with room; a bfloat16 result adds 2^-9 of itself.  The gated
product multiplies two such sums, silu by a fast exponential: 2^-6 of the product of their sizes in bfloat16."""
import math

import pytest
import torch

from plain_lowbit import e4m3, product8, rounded8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F = torch.float64


def K():
    from exl3_server_b200.ops import kernels
    return kernels


def make(M, N, Kd, seed=0, x_scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(M, Kd, device=DEV, generator=g) * x_scale * torch.exp(torch.randn(1, Kd, device=DEV, generator=g))).bfloat16()
    w, s = K().fp8_quantize_weight((torch.randn(N, Kd, device=DEV, generator=g) * 0.05).bfloat16())
    return x, w, s


def sizes(x, w, s):
    """sum |x| |w| of the rounded values."""
    return product8(x.abs(), w.float().abs(), s)


@pytest.mark.parametrize("M,Kd", [(1, 16), (3, 128), (17, 144), (130, 1000 // 16 * 16), (5, 4096)])
def test_rounding_is_exact(M, Kd):
    g = torch.Generator(device=DEV).manual_seed(M)
    wide = (torch.randn(M, Kd + 24, device=DEV, generator=g) * 5).bfloat16()
    x = wide[:, 8:8 + Kd]
    x[0, :min(16, Kd)] = 0
    codes, scales = K().fp8_quantize(x)
    want_c, want_s = rounded8(x)
    assert torch.equal(codes.float().to(F), want_c) and torch.equal(scales.to(F), want_s)


def test_rounding_of_extremes():
    x = torch.zeros(6, 256, device=DEV).bfloat16()
    x[1, 3], x[2, 5], x[3, 130] = math.nan, math.inf, 3e38
    x[4, 7] = 1e-38
    x[5] = 1.0
    codes, scales = K().fp8_quantize(x)
    c = codes.float()
    assert bool((c[0] == 0).all()) and bool((scales[0] > 0).all())
    assert bool(c[1, 3].isnan()) and bool(c[1, 128:].isfinite().all()) and bool(c[2, 5].isnan()) and not math.isfinite(float(scales[2, 0]))
    assert float(c[3, 130]) == 448.0 and float(c[5, 0]) == 448.0 and bool(c[4].isfinite().all())


@pytest.mark.parametrize("N,Kd", [(128, 128), (130, 256), (257, 144), (64, 1040)])
def test_weights_rounding(N, Kd):
    g = torch.Generator(device=DEV).manual_seed(N)
    w = (torch.randn(N, Kd, device=DEV, generator=g) * torch.exp(torch.randn(N, 1, device=DEV, generator=g))).bfloat16()
    codes, scales = K().fp8_quantize_weight(w)
    assert scales.shape == (-(-N // 128), -(-Kd // 128))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = w[128 * i:128 * i + 128, 128 * j:128 * j + 128].float()
            a = b.abs().max()
            assert float(scales[i, j]) == float(a / torch.tensor(448.0, device=DEV))
            assert torch.equal(codes[128 * i:128 * i + 128, 128 * j:128 * j + 128].float().to(F), e4m3(b * (torch.tensor(448.0, device=DEV) / a)))
    host, host_s = K().fp8_quantize_weight(w.cpu())
    assert torch.equal(host.float(), codes.float().cpu()) and torch.equal(host_s, scales.cpu())


ROWS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 129, 256, 257, 300]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("N,Kd", [(128, 128), (200, 272), (333, 1040), (2304, 144), (272, 16), (1000, 2304)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_product(M, N, Kd, out_dtype):
    x, w, s = make(M, N, Kd, seed=M + N)
    bias = torch.randn(N, device=DEV).bfloat16() if (M + N) % 2 else None
    y = K().fp8_linear(x, w, s, bias=bias, out_dtype=out_dtype)
    want, size = product8(x, w, s, bias), sizes(x, w, s)
    assert y.dtype == out_dtype and y.shape == (M, N)
    bound = 2.0 ** -17 * size + (2.0 ** -8 * want.abs() if out_dtype == torch.bfloat16 else 2.0 ** -22 * want.abs()) + 1e-30
    assert bool(((y.to(F) - want).abs() <= bound).all()), float(((y.to(F) - want).abs() / bound).max())
    K().check_status()


@pytest.mark.parametrize("M", [1, 16, 40, 64, 130, 300])
@pytest.mark.parametrize("N,Kd", [(16, 128), (272, 272), (4096, 1040)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_gated_product(M, N, Kd, out_dtype):
    x, w, s = make(M, N, Kd, seed=M + N + 1, x_scale=0.5)
    y = K().fp8_linear(x, w, s, out_dtype=out_dtype, gated=True)
    want = product8(x, w, s, gated=True)
    z, size = product8(x, w, s).view(M, N // 16, 2, 8), sizes(x, w, s).view(M, N // 16, 2, 8)
    gate, up = z[:, :, 0], z[:, :, 1]
    # d(silu) <= 1.1 per unit of the gate; a fast exponential and division: a few 2^-21
    bound = (2.0 ** -17 * (1.1 * size[:, :, 0] * up.abs() + gate.abs() * size[:, :, 1])).reshape(M, N // 2) + \
        (2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -18) * want.abs() + 1e-7
    assert y.shape == (M, N // 2) and bool(((y.to(F) - want).abs() <= bound).all())


def test_rows_do_not_depend_on_each_other():
    x, w, s = make(64, 700, 2304, seed=3)
    k = K()
    some = k.fp8_linear(x[:16], w, s, out_dtype=torch.float32)
    assert all(torch.equal(k.fp8_linear(x[i:i + 1], w, s, out_dtype=torch.float32), some[i:i + 1]) for i in (0, 7, 15))
    many = k.fp8_linear(x, w, s, out_dtype=torch.float32)
    assert torch.equal(k.fp8_linear(x[:40], w, s, out_dtype=torch.float32), many[:40])
    assert torch.equal(many[:16], some)


@pytest.mark.parametrize("M", [5, 50, 400])
def test_rows_that_are_not_finite_stay_by_themselves(M):
    x, w, s = make(M, 300, 400, seed=4)
    k = K()
    clean = k.fp8_linear(x, w, s)
    x[1, 7], x[3, 399] = math.nan, -math.inf
    y = k.fp8_linear(x, w, s)
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().all())
    rest = [i for i in range(M) if i not in (1, 3)]
    assert torch.equal(y[rest], clean[rest])


def test_rows_apart_and_another_stream():
    k = K()
    x, w, s = make(70, 384, 512, seed=5)
    wide = torch.zeros(70, 600, device=DEV, dtype=torch.bfloat16)
    wide[:, 40:552] = x
    for m in (3, 70):
        want = k.fp8_linear(x[:m], w, s)
        assert torch.equal(k.fp8_linear(wide[:m, 40:552], w, s), want)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = k.fp8_linear(x[:m], w, s)
        torch.cuda.current_stream().wait_stream(st)
        assert torch.equal(got, want)
    assert k.fp8_linear(x[:0], w, s).shape == (0, 384)


def test_refusals():
    from exl3_server_b200.ops.lib import KernelLibraryError as E
    k = K()
    x, w, s = make(4, 160, 256)
    for f in (
        lambda: k.fp8_linear(x.float(), w, s),
        lambda: k.fp8_linear(x[:, :248], w[:, :248].contiguous(), s),                    # 248 features
        lambda: k.fp8_linear(x, w[:, :128].contiguous(), s),
        lambda: k.fp8_linear(x, w.float(), s),
        lambda: k.fp8_linear(x, w, s[:1]),
        lambda: k.fp8_linear(x, w, s.double()),
        lambda: k.fp8_linear(x, w, s, bias=torch.zeros(160, device=DEV)),
        lambda: k.fp8_linear(x, w, s, bias=torch.zeros(160, device=DEV).bfloat16(), gated=True),
        lambda: k.fp8_linear(x, w[:152].contiguous(), s, gated=True),
        lambda: k.fp8_linear(x, w, s, out_dtype=torch.float16),
        lambda: k.fp8_linear(x, w, s, out=torch.empty(4, 100, device=DEV).bfloat16()),
        lambda: k.fp8_linear(x.cpu(), w, s),
        lambda: k.fp8_quantize(x.float()),
        lambda: k.fp8_quantize(x[:, :8]),
        lambda: k.fp8_quantize_weight(w[0]),
    ):
        with pytest.raises(E):
            f()
