"""Products in 8-bit floating point whose weights were written by the kernel just ahead in the stream, and rows that lie anywhere."""
import pytest
import torch

from test_fp8_gpu import DEV, K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fixed_order", [True, False])
@pytest.mark.parametrize("M", [1, 8, 40])
def test_weights_that_have_just_been_rounded(M, fixed_order):
    """The codes and scales of one row are those of a weight with one output feature; other values in the same memory each time."""
    k, Kd = K(), 8192
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, Kd, device=DEV, generator=g).bfloat16()
    rows = [torch.randn(1, Kd, device=DEV, generator=g).bfloat16() for _ in range(40)]
    want = []
    for r in rows:
        codes, scales = k.fp8_quantize(r)
        torch.cuda.synchronize()
        want.append(k.fp8_linear(x, codes, scales, fixed_order=fixed_order))
    torch.cuda.synchronize()
    got = [k.fp8_linear(x, *k.fp8_quantize(r), fixed_order=fixed_order) for r in rows]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("fixed_order", [True, False])
@pytest.mark.parametrize("stride", [257, 300])
def test_one_row_of_a_matrix_with_any_stride(stride, fixed_order):
    """A matrix of one row has no distance between rows, whatever its stride says."""
    k = K()
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(1, 256, device=DEV, generator=g).bfloat16()
    w, s = k.fp8_quantize_weight(torch.randn(160, 256, device=DEV, generator=g).bfloat16())
    odd = torch.zeros(1, stride, device=DEV).bfloat16()
    odd[:, :256] = x
    assert odd[:, :256].stride(0) == stride
    assert torch.equal(k.fp8_linear(odd[:, :256], w, s, fixed_order=fixed_order), k.fp8_linear(x, w, s, fixed_order=fixed_order))
    for a, b in zip(k.fp8_quantize(odd[:, :256]), k.fp8_quantize(x)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
