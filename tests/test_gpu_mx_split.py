"""4-bit products whose last rows run in another kernel than the first ones: 256 x 256 tiles for whole
rounds, then 128 x 128 tiles or the kernel of few rows, with row origins, scales and results that
count from the whole product's first row.  test_mx_plan.py checks that each size here is dealt out as it says."""
import pytest
import torch

from icsa_hip import mx_linear, mx_quantize
from test_gpu_mx import _linear_case, _x

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# M, N, K, token tiles (of 256 rows) of the first kernel, kernel of the other rows
SPLITS = [(9360, 2000, 1300, 32, "tiles"), (3120, 5120, 4352, 12, "rows"), (17003, 1001, 1300, 64, "tiles"),
          (3081, 5120, 4352, 12, "rows")]


@pytest.mark.parametrize("M,N,K,first,rest", SPLITS)
@pytest.mark.parametrize("out_dtype,act,bias", [(BF, "gelu_tanh", torch.float32), (torch.float32, None, BF)])
def test_last_rows_in_another_kernel(gpu, M, N, K, first, rest, out_dtype, act, bias):
    print(f"[mx] split {M}x{N}x{K} {out_dtype} {act}", flush=True)
    _linear_case(gpu, M, N, K, BF, out_dtype, act, bias, M + N)


@pytest.mark.parametrize("M,N,K,first,rest", SPLITS)
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_last_rows_into_4_bits(gpu, M, N, K, first, rest, act):
    """Codes and scales of the whole product: those of its f32 result, which test_last_rows_in_another_kernel compares
    with float64.  Both calls deal the rows out alike, so their f32 sums are the same numbers."""
    print(f"[mx] split {M}x{N}x{K} to 4 bits {act}", flush=True)
    g = torch.Generator().manual_seed(M)
    x, w = mx_quantize(_x(M, K, BF, 1, 0.7).to(gpu)), mx_quantize((_x(N, K, torch.float32, 2, 0.3) / K ** 0.5).to(gpu))
    b = torch.randn(N, generator=g).to(gpu)
    y = mx_linear(x, w, b, act, "mxfp4")
    z = mx_quantize(mx_linear(x, w, b, act, torch.float32))
    assert torch.equal(y.codes, z.codes) and torch.equal(y.scales, z.scales)
