"""The 4-bit quantisation and product on the GPU against float64 (oracle.mxfp4).

Codes and scales are whole numbers and have to be equal.  A product's tolerance: products of two
e2m1 values are exact in f32, so a result is off by its additions, at most K steps of 2^-23 (a
truncating adder's) of sum |x w|, by the bias and activation (a few f32 steps of their inputs; GELU's
slope is at most 1.13), and by the rounding to its type, eps / 2 of the value.
"""
import math

import pytest
import torch

from icsa_hip import MXFP4Tensor, mx_linear, mx_quantize
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _x(M, K, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, K, generator=g) * torch.exp(spread * torch.randn(M, K // 7 + 1, generator=g))
            .repeat_interleave(7, 1)[:, :K]).to(dtype)


def _check_quantized(t, x):
    codes, scales = O.quantize(x)
    assert torch.equal(t.scales.cpu(), scales)
    assert torch.equal(t.codes.cpu(), codes)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 255), (4, 256), (7, 257), (1, 5120), (33, 511),
                                 (65, 1000), (130, 4100), (2, 13824)])
def test_quantize_and_back(gpu, M, K, dtype):
    print(f"[mx] quantize {M}x{K} {dtype}", flush=True)
    x = _x(M, K, dtype, M + K)
    t = mx_quantize(x.to(gpu))
    _check_quantized(t, x)
    v = O.values(t.codes, t.scales, K)
    assert torch.equal(t.dequantize(torch.float32).cpu().double(), v)
    assert torch.equal(t.dequantize().cpu().double(), v)


def test_quantize_borders(gpu):
    """Every tie and its neighbours, both signs, at scales over the whole range of exponents, and
    amax at powers of two."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.984375], dtype=torch.float32)
    near = torch.cat([mids, torch.nextafter(mids, torch.zeros(())), torch.nextafter(mids, torch.full((), 9.0))])
    row = torch.cat([near, torch.tensor([4.0, -4.0])])                      # amax in [4, 8): scale 1
    rows = torch.stack([torch.ldexp(row, torch.tensor(e)) for e in range(-120, 126, 3)])
    rows = torch.cat([rows, -rows])
    t = mx_quantize(rows.to(gpu))
    _check_quantized(t, rows)


def test_quantize_small_large_and_not_finite(gpu):
    x = torch.zeros(12, 64)
    x[1, :32] = 2.0 ** -149                               # the least f32
    x[2, :32] = 2.0 ** -126
    x[2, 5] = 3.0 * 2.0 ** -127
    x[3, 7] = -torch.finfo(torch.float32).max
    x[4, 3] = math.nan
    x[5, 40] = math.inf
    x[6, 0], x[6, 31] = -math.inf, 1.0
    x[7, :] = torch.finfo(torch.float32).min
    x[8, :32] = 1e-40
    x[9, :] = -0.0
    x[10, :32] = 2.0 ** -128 * 1.5
    x[11, ::2] = 2.0 ** -125
    t = mx_quantize(x.to(gpu))
    _check_quantized(t, x)
    v = O.values(t.codes, t.scales, 64)
    for dt in (torch.float32, BF):
        assert torch.equal(torch.nan_to_num(t.dequantize(dt).cpu().double(), nan=1e300), torch.nan_to_num(v, nan=1e300))


def test_quantize_strides_and_shapes(gpu):
    base = _x(24, 700, BF, 5).to(gpu)
    for v in (base[:, 3:603], base[::2, :640], base[:, ::2], base.t(), base.view(2, 3, 4, 700)[:, 1, :, 1:302]):
        t = mx_quantize(v)
        assert t.shape == v.shape
        _check_quantized(t, v.reshape(-1, v.shape[-1]).cpu())
    one = mx_quantize(base[0])
    assert one.shape == (700,) and one.dequantize().shape == (700,)
    none = mx_quantize(base[:0])
    assert none.shape == (0, 700) and none.dequantize().shape == (0, 700)


def _tolerance(x64, w64, ref, dtype, bias):
    K = x64.shape[1]
    mass = x64.abs() @ w64.abs().t()
    inner = (K + 4) * 2.0 ** -23 * mass + 2.0 ** -22 * (bias.abs() + ref.abs())
    eps = {BF: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    return 1.13 * inner * (1 + eps) + eps * ref.abs() + 1e-37


def _linear_case(gpu, M, N, K, x_dtype, out_dtype, act, bias_dtype, seed=0):
    x = _x(M, K, x_dtype, seed, 0.7)
    w = _x(N, K, torch.float32, seed + 1, 0.3) / math.sqrt(K)
    g = torch.Generator().manual_seed(seed + 2)
    b = None if bias_dtype is None else torch.randn(N, generator=g).to(bias_dtype)
    wq = mx_quantize(w.to(gpu))
    y = mx_linear(x.to(gpu), wq, None if b is None else b.to(gpu), activation=act, out_dtype=out_dtype)
    x64 = O.values(*O.quantize(x), K)
    w64 = O.values(wq.codes, wq.scales, K)
    bias = torch.zeros(N).double() if b is None else b.double()
    ref = x64 @ w64.t() + bias
    if act:
        ref = O.gelu_tanh(ref)
    assert y.shape == (M, N) and y.dtype == out_dtype
    d = (y.double().cpu() - ref).abs()
    tol = _tolerance(x64, w64, ref, out_dtype, bias)
    assert (d <= tol).all(), f"{(d / tol).max().item():.2f} of the tolerance, {d.max().item():.3e}"


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 64), (1, 5120, 5120), (2, 33, 300), (7, 130, 511), (16, 64, 256),
                                   (31, 257, 1000), (32, 100, 768), (33, 96, 512), (64, 256, 1024), (65, 129, 257),
                                   (100, 300, 2048), (127, 640, 640), (128, 128, 256), (257, 513, 1300), (512, 1280, 512),
                                   (1000, 1000, 1000)])
@pytest.mark.parametrize("out_dtype,act,bias", [(BF, None, torch.float32), (torch.float32, "gelu_tanh", BF), (BF, "gelu_tanh", None)])
def test_linear(gpu, M, N, K, out_dtype, act, bias):
    print(f"[mx] linear {M}x{N}x{K} {out_dtype} {act}", flush=True)
    _linear_case(gpu, M, N, K, BF if M % 2 else torch.float32, out_dtype, act, bias, M + N)


def test_linear_large_tiles(gpu):
    """Sizes that take the large tile, whole and ragged, with several tiles a workgroup; sizes whose last rows go to
    smaller tiles or to the kernel of few rows; one group of k."""
    for M, N, K in ((4096, 4096, 512), (4099, 4110, 300), (3120, 5120, 1300), (9360, 2000, 1000), (4660, 4000, 900), (5000, 4500, 200)):
        print(f"[mx] large {M}x{N}x{K}", flush=True)
        _linear_case(gpu, M, N, K, BF, BF, None, torch.float32, M)


@pytest.mark.parametrize("M,N,K", [(1, 40, 256), (3, 256, 300), (33, 300, 512), (130, 1000, 257), (4100, 4097, 256)])
def test_linear_into_4_bits(gpu, M, N, K):
    """A result in 4 bits is the quantisation of the f32 result: its scale is that of the true amax, or a
    neighbour where amax is within the product's error of a power of two, and its codes' values are
    within half a code step of the true value."""
    print(f"[mx] to 4 bits {M}x{N}x{K}", flush=True)
    x, w = _x(M, K, BF, 1, 0.7), _x(N, K, torch.float32, 2, 0.3) / math.sqrt(K)
    wq, xq = mx_quantize(w.to(gpu)), mx_quantize(x.to(gpu))
    b = torch.randn(N)
    y = mx_linear(xq, wq, b.to(gpu), activation="gelu_tanh", out_dtype="mxfp4")
    f = mx_linear(xq, wq, b.to(gpu), activation="gelu_tanh", out_dtype=torch.float32)
    _check_quantized(y, f.cpu())              # the same f32 results, rounded to codes: equal
    assert isinstance(y, MXFP4Tensor) and y.shape == (M, N)


def test_two_layers(gpu):
    """Quantise, product with GELU into 4 bits, product: the hidden codes may differ from float64's
    where a value is within the f32 error of a border; one code step of one hidden value moves an output by
    at most that step times the weight, far below the bf16 rounding of sums of 1,000 terms."""
    M, K, N = 70, 300, 1000
    x, w1 = _x(M, K, BF, 3, 0.5), _x(N, K, torch.float32, 4, 0.3) / math.sqrt(K)
    w2 = _x(K, N, torch.float32, 5, 0.3) / math.sqrt(N)
    w1q, w2q = mx_quantize(w1.to(gpu)), mx_quantize(w2.to(gpu))
    h = mx_linear(x.to(gpu), w1q, activation="gelu_tanh", out_dtype="mxfp4")
    y = mx_linear(h, w2q)
    h64 = O.values(h.codes, h.scales, N)
    ref = h64 @ O.values(w2q.codes, w2q.scales, N).t()
    d = (y.double().cpu() - ref).abs()
    assert (d <= _tolerance(h64, O.values(w2q.codes, w2q.scales, N), ref, BF, torch.zeros(K).double())).all()


def test_not_finite_rows_stay_apart(gpu):
    """A NaN or an infinity of one row reaches that row alone, and a NaN weight row its output alone."""
    for M in (5, 200):
        x = _x(M, 512, torch.float32, 6, 0.5)
        x[1, 100], x[3, 5] = math.nan, math.inf
        w = _x(300, 512, torch.float32, 7, 0.3)
        w[17, 3] = math.nan
        y = mx_linear(x.to(gpu), mx_quantize(w.to(gpu)), out_dtype=torch.float32).cpu()
        bad = torch.zeros(M, 300, dtype=torch.bool)
        bad[1], bad[3], bad[:, 17] = True, True, True
        assert torch.equal(torch.isnan(y), bad)


def test_rows_far_apart(gpu):
    """Rows behind 32-bit offsets, of the values, the codes and the results, equal the same rows on their own.  A row's
    sums do not depend on the tile it is in (steps of k in order in every tile)."""
    big = torch.zeros(9001, 1 << 18, dtype=BF, device=gpu)
    x = big[:, 1000:1600]
    x.normal_()
    a, b = mx_quantize(x), mx_quantize(x.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    a, b = mx_quantize(big), mx_quantize(big[-70:])
    assert torch.equal(a.codes[-70:], b.codes) and torch.equal(a.scales[:, -70:], b.scales)
    del big, x, a, b
    x = torch.randn(70001, 256, device=gpu).to(BF)
    w = mx_quantize(torch.randn(32776, 256, device=gpu) / 16)
    bias = torch.randn(32776, device=gpu)
    assert torch.equal(mx_linear(x, w, bias)[-300:], mx_linear(x[-300:], w, bias))
    y, z = (mx_linear(t, w, bias, "gelu_tanh", "mxfp4") for t in (x, x[-300:]))
    assert torch.equal(y.codes[-300:], z.codes) and torch.equal(y.scales[:, -300:], z.scales)
    assert torch.equal(y.dequantize(torch.float32)[-300:], z.dequantize(torch.float32))


@pytest.mark.parametrize("M,N,K", [(300, 700, 600), (4099, 4110, 300), (9360, 2001, 520)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_bias_of_either_type_and_any_start(gpu, M, N, K, dtype):
    """Over several tiles a workgroup, ragged ends, a bias that starts behind another tensor's first element: the result is
    that without a bias, of the same f32 sums, and the bias (an f32 addition at another place: K + 2 steps of 2^-24 at most)."""
    print(f"[mx] bias {M}x{N}x{K} {dtype}", flush=True)
    x, w = mx_quantize(_x(M, K, BF, 1, 0.7).to(gpu)), mx_quantize((_x(N, K, torch.float32, 2, 0.3) / math.sqrt(K)).to(gpu))
    b = torch.randn(N + 1, generator=torch.Generator().manual_seed(3)).to(dtype).to(gpu)[1:]
    plain = mx_linear(x, w, None, out_dtype=torch.float32).double()
    y = mx_linear(x, w, b, out_dtype=torch.float32).double()
    mass = mx_linear(mx_quantize(x.dequantize().abs()), mx_quantize(w.dequantize().abs()), None, out_dtype=torch.float32).double()
    assert ((y - plain - b.double()).abs() <= 2.0 ** -24 * (K + 2) * (1.01 * mass + b.double().abs())).all()
