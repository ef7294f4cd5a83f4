"""The int8 product against 64-bit arithmetic: the codes are whole numbers and equal, the sums are exact, what is left is the
conversion of the sum to FP32 and two products by scales (three roundings of 2^-24) and the rounding to the output's type: half a
step of the value, or half of the type's smallest step below its normal numbers (FP16: 2^-25)."""

import math

import pytest

from mylocal_llm_b200 import _lib, Int8Weight, int8_linear, int8_matmul, packed_to_device, quantize_int8_rows
from mylocal_llm_b200.quantize import quantize

pytestmark = pytest.mark.gpu


def quantised(torch, x):
    scale = (x.double().abs().amax(-1) / 127).float().clamp_min(2.0 ** -126)
    return (x.double() / scale.double()[:, None]).round().to(torch.int8), scale


def check(torch, y, codes, scales, weight, k):
    want = codes[:, :k].double() @ weight.codes[:, :k].double().t() * scales.double()[:, None] * weight.scales.double()
    kind = torch.finfo(y.dtype)
    bound = (3 * 2.0 ** -24 + kind.eps / 2 * 1.01) * want.abs() + kind.tiny * kind.eps / 2
    assert torch.isfinite(y).all()
    assert ((y.double() - want).abs() <= bound).all()


def random_weight(torch, n, k, gen):
    codes = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=gen)
    return Int8Weight(codes, torch.rand(n, device="cuda", generator=gen) * 1e-3 + 1e-4)


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (2, 16), (5, 17), (4, 255), (7, 2048), (2, 8191), (3, 20000), (300, 1030)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_quantised_rows_equal_the_definition(cuda, rows, k, dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows + k)
    x = (torch.randn(rows, k, device="cuda", generator=gen) * torch.exp(3 * torch.randn(rows, 1, device="cuda", generator=gen))).to(getattr(torch, dtype))
    x[rows // 2] = 0
    codes, scales = quantize_int8_rows(x)
    want, scale = quantised(torch, x)
    assert torch.equal(codes[:, :k], want) and torch.equal(scales, scale) and not codes[:, k:].any()
    wide = torch.zeros(rows, k + 5, dtype=x.dtype, device="cuda")
    wide[:, 3:3 + k] = x
    odd, again = quantize_int8_rows(wide[:, 3:3 + k])                   # rows at any address
    assert torch.equal(odd, codes) and torch.equal(again, scales)


def test_quantised_rows_at_borders_and_beyond(cuda):
    torch = cuda
    x = torch.zeros(7, 300, device="cuda")
    x[0] = torch.arange(300, device="cuda") * 0.5 - 74.75
    x[0, 0] = 127.0                                                     # scale 1: k + 1/2 and k + 1/4
    x[1, 5] = 2.0 ** -130                                               # below the smallest scale
    x[2, :3] = torch.tensor([2.0 ** -126, -2.0 ** -126 * 0.5, 2.0 ** -126 * 1.5])
    x[3, :2] = torch.tensor([3.0e38, -1.5e38])
    x[4, 7], x[5, 8], x[6, 9] = math.nan, math.inf, -math.inf
    codes, scales = quantize_int8_rows(x)
    want, scale = quantised(torch, x[:4])
    assert torch.equal(codes[:4, :300], want) and torch.equal(scales[:4], scale)
    assert torch.isnan(scales[4:]).all()
    y = int8_linear(x, Int8Weight(torch.ones(3, 300, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")))
    assert torch.isfinite(y[:4]).all() and torch.isnan(y[4:]).all()


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 128, 128), (2, 7, 100), (1, 8192, 2048), (3, 250, 16), (8, 4096, 4096), (16, 333, 2049), (17, 129, 640), (33, 2000, 1000),
    (64, 512, 128), (65, 640, 3000), (100, 1003, 777), (128, 256, 512), (129, 4100, 2100), (257, 300, 130), (500, 1111, 4099), (1000, 2048, 512),
    (2049, 515, 260)])
def test_products_equal_64_bits(cuda, m, n, k):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    weight = random_weight(torch, n, k, gen)
    x = torch.randn(m, k, device="cuda", generator=gen)
    codes, scales = quantize_int8_rows(x)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        check(torch, int8_matmul(codes, scales, weight, out_dtype=out), codes, scales, weight, k)
    assert torch.equal(int8_linear(x, weight), int8_matmul(codes, scales, weight))
    assert torch.equal(int8_matmul(codes, scales, weight), int8_matmul(codes, scales, weight))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_sums_at_the_limit_of_32_bits(cuda, m):
    torch = cuda
    k = 131071
    weight = Int8Weight(torch.full((130, k), -127, dtype=torch.int8, device="cuda"), torch.ones(130, device="cuda"))
    codes = torch.full((m, 131072), 127, dtype=torch.int8, device="cuda")
    scales = torch.full((m,), 2.0 ** -20, device="cuda")
    y = int8_matmul(codes, scales, weight)
    assert (y == torch.tensor(-127.0 * 127 * k, dtype=torch.float64).float().cuda() * 2.0 ** -20).all()
    with pytest.raises(NotImplementedError):
        Int8Weight(torch.ones(1, 131072, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))


def test_what_lies_behind_k_does_not_count(cuda):
    """Codes behind K are zero in one of the operands: whatever the other holds there has no effect, nor has memory behind the
    last row."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(0)
    for m, n, k in ((3, 5, 21), (40, 140, 133), (300, 200, 70)):
        weight = random_weight(torch, n, k, gen)
        x = torch.randn(m, k, device="cuda", generator=gen)
        codes, scales = quantize_int8_rows(x)
        want = int8_matmul(codes, scales, weight)
        codes[:, k:] = 99
        assert torch.equal(int8_matmul(codes, scales, weight), want)


def test_leading_dimensions_types_and_empty_batches(cuda):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(1)
    weight = Int8Weight.quantize(torch.randn(48, 96, device="cuda", generator=gen).to(torch.bfloat16))
    x = torch.randn(2, 3, 96, device="cuda", generator=gen).half()
    y = int8_linear(x, weight)
    assert y.shape == (2, 3, 48) and y.dtype == torch.float16
    assert torch.equal(y.reshape(6, 48), int8_linear(x.reshape(6, 96), weight))
    assert int8_linear(x[:0], weight).shape == (0, 3, 48)
    assert weight.nbytes == 48 * 96 + 4 * 48


@pytest.mark.parametrize("fmt", ["Q8_0", "Q4_K"])
def test_weights_from_packed_matrices(cuda, fmt):
    """Within the rounding of the weights (half a step of max / 127) of the packed projection."""
    torch = cuda
    import numpy as np
    from mylocal_llm_b200.quantized_linear import dequantize_device
    packed = packed_to_device(quantize(np.random.default_rng(0).normal(0, 0.02, (130, 512)).astype(np.float32), fmt))
    weight = Int8Weight.from_packed(packed)
    dense = dequantize_device(packed.data, 130, 512, packed.quant_type)
    off = (weight.codes[:, :512].double() * weight.scales.double()[:, None] - dense.double()).abs()
    assert (off <= weight.scales.double()[:, None] * 0.5000001).all()


def test_refusals(cuda):
    torch = cuda
    weight = Int8Weight(torch.ones(4, 40, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))
    x = torch.randn(3, 40, device="cuda")
    codes, scales = quantize_int8_rows(x)
    with pytest.raises(ValueError):
        int8_linear(torch.randn(3, 41, device="cuda"), weight)
    with pytest.raises(ValueError):
        int8_matmul(codes[:, :40], scales, weight)
    with pytest.raises(ValueError):
        int8_matmul(codes, scales[:2], weight)
    with pytest.raises(ValueError):
        int8_matmul(codes.float(), scales, weight)
    with pytest.raises(TypeError):
        int8_matmul(codes, scales, weight.codes)
    with pytest.raises(TypeError):
        int8_matmul(codes, scales, weight, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        quantize_int8_rows(x.double())
    with pytest.raises(ValueError):
        quantize_int8_rows(x.t())
    with pytest.raises(ValueError):
        Int8Weight(torch.ones(4, 40, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"))
    with pytest.raises(ValueError):
        Int8Weight(torch.ones(4, 40, device="cuda"), torch.ones(4, device="cuda"))
    with pytest.raises(TypeError):
        Int8Weight.from_packed(x)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,k,stride", [(9, 1, 1), (9, 7, 9), (5, 1023, 1023), (40, 300, 307), (3, 4100, 4101), (700, 33, 41), (4, 8200, 8203), (2, 20001, 20002)])
def test_rows_at_every_offset_among_what_does_not_count(cuda, rows, k, stride, dtype):
    """Rows that begin at every element of 16 bytes; NaN and infinities before, between and behind them."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows + k)
    for first in range(9):
        flat = torch.full((first + rows * stride + 9,), math.nan, dtype=getattr(torch, dtype), device="cuda")
        flat[::2] = math.inf
        x = flat[first:first + rows * stride].view(rows, stride)[:, :k]
        x.copy_(torch.randn(rows, k, device="cuda", generator=gen))
        codes, scales = quantize_int8_rows(x)
        want, scale = quantised(torch, x)
        assert torch.equal(codes[:, :k], want) and torch.equal(scales, scale) and not codes[:, k:].any()


@pytest.mark.parametrize("m,n,k", [(130, 8231, 300), (1262, 4099, 200), (300, 9000, 17), (257, 16383, 129), (32, 77, 64), (31, 4001, 128)])
def test_rows_of_outputs_at_any_alignment(cuda, m, n, k):
    """Outputs whose rows are not 16-byte aligned, and nothing written behind the last row."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    weight = random_weight(torch, n, k, gen)
    codes, scales = quantize_int8_rows(torch.randn(m, k, device="cuda", generator=gen))
    for dtype, ident in ((torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)):
        for first in (0, 1, 3):
            flat = torch.full((first + m * n + 64,), 77.0, dtype=dtype, device="cuda")
            y = flat[first:first + m * n].view(m, n)
            _lib.call("b200q_int8_gemm", weight.codes.data_ptr(), weight.codes.shape[1], weight.scales.data_ptr(), n, k, codes.data_ptr(),
                      codes.shape[1], scales.data_ptr(), m, y.data_ptr(), ident, torch.cuda.current_stream().cuda_stream)
            check(torch, y, codes, scales, weight, k)
            assert (flat[:first] == 77).all() and (flat[first + m * n:] == 77).all()
