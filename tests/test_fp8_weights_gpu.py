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
