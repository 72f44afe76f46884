"""The 4-bit product at the ends of the exponents' range, and biases that are not finite."""
import math

import pytest
import torch

from icsa_hip import mx_linear, mx_quantize
from test_gpu_mx import _x

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("M,N,K", [(1, 40, 300), (40, 130, 520), (300, 260, 1000), (9360, 2000, 1300)])
def test_powers_of_two_pass_through(gpu, M, N, K):
    """Factors of 2^a on x and 2^b on the weights change no code and no mantissa: the f32 results are 2^(a + b) times as large,
    bit for bit, where they and their terms stay normal numbers (terms here: 2^-20 to 2^12 at a + b = 0)."""
    print(f"[mx range] {M}x{N}x{K}", flush=True)
    x, w = _x(M, K, torch.float32, 1, 0.3).clamp(-8, 8).to(gpu), _x(N, K, torch.float32, 2, 0.3).clamp(-8, 8).to(gpu)
    x, w = (torch.where(t.abs() < 2.0 ** -6, 2.0 ** -6, t) for t in (x, w))
    plain = mx_linear(x, mx_quantize(w), out_dtype=torch.float32)
    for a, b in ((-118, 112), (118, -118), (-110, 10), (60, 40), (-50, -50), (110, 0)):
        y = mx_linear(torch.ldexp(x, torch.tensor(a)), mx_quantize(torch.ldexp(w, torch.tensor(b))), out_dtype=torch.float32)
        assert torch.equal(y, torch.ldexp(plain, torch.tensor(a + b))), (a, b)


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_biases_that_are_not_finite(gpu, M, act):
    """Each reaches its own output: GELU(inf) is inf, GELU(-inf) by its formula -inf * 0, not a number."""
    x, w = _x(M, 300, BF, 3, 0.3).to(gpu), mx_quantize(_x(200, 300, torch.float32, 4, 0.3).to(gpu))
    b = torch.zeros(200, device=gpu)
    want = mx_linear(x, w, b, act, torch.float32)
    b[7], b[100], b[199], b[31], b[32] = math.inf, -math.inf, math.nan, 3e38, -3e38
    y = mx_linear(x, w, b, act, torch.float32)
    want[:, 7], want[:, 199], want[:, 31] = math.inf, math.nan, 3e38
    want[:, 100], want[:, 32] = (math.nan, -0.0) if act else (-math.inf, -3e38)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(y, nan=0.0, posinf=1e30, neginf=-1e30).clamp(-1e30, 1e30),
                       torch.nan_to_num(want, nan=0.0, posinf=1e30, neginf=-1e30).clamp(-1e30, 1e30))
