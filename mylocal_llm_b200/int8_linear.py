"""Projections in 8-bit integers: int8 weights with one scale per output channel, activations quantised per token.

Opt-in like the Q8_1 mode (``q8_1.py``, ``mini_llm/ops/mixed_q8_gpu.py:203-251`` of the reference), of which it is the
whole-row form: one scale for a token's K activations and one for a channel's K weights, so that the K products are summed as
exact 32-bit integers on the tensor cores and scaled once at the end. The result differs from the product of the unquantised
operands by the rounding of both to int8 (half a step of max / 127 per element).

    weight = Int8Weight.quantize(dense)                 # or Int8Weight.from_packed(device_packed_weight)
    y = int8_linear(x, weight)                          # x [..., K] FP32 / FP16 / BF16 -> [..., N]
"""

from . import _lib
from .kv8_cache import _dtype_id, _launch
from .quantized_linear import DevicePackedGGUFWeight, dequantize_device

INT8_MAX_K = 131071         # so many products of two codes fit a 32-bit sum
INT8_MAX_SIZE = 2 ** 30     # rows or columns of a matrix


def _torch():
    import torch
    return torch


def quantize_int8_rows(x):
    """``x`` ``[..., K]`` (FP32 / FP16 / BF16 CUDA tensor) -> (int8 codes ``[rows, K']``, FP32 scales ``[rows]``): scale = max |x| /
    127 of the row (at least 2^-126), codes = x / scale to the nearest integer, ties to even; K' is K rounded up to a multiple of
    16 and the codes behind K are zero. A row with a NaN or an infinity has the scale NaN."""
    return _quantize(x, 0)


def _quantize(x, early):
    torch = _torch()
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError("quantize_int8_rows expects a torch CUDA tensor")
    ident = _dtype_id(x, "x")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one element")
    k = x.shape[-1]
    if x.ndim == 2 and x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= k):
        rows, x_row = x.shape[0], (x.stride(0) if x.shape[0] > 1 else k)
    elif x.is_contiguous():
        rows, x_row = x.numel() // k, k
    else:
        raise ValueError("x must be contiguous, or two-dimensional with rows of consecutive elements")
    if max(rows, k) > INT8_MAX_SIZE:
        raise NotImplementedError(f"at most {INT8_MAX_SIZE} rows and columns")
    padded = -(-k // 16) * 16
    codes = torch.empty((rows, padded), dtype=torch.int8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows:
        _launch(x.device, "b200q_int8_quantize", x.data_ptr(), ident, rows, k, x_row, codes.data_ptr(), padded, scales.data_ptr(), early)
    return codes, scales


class Int8Weight:
    """An int8 matrix ``[N, K]`` with FP32 scales ``[N]`` (value = code * scale). ``codes`` is kept with rows of a multiple of 16
    bytes (a copy is made where K is none)."""

    def __init__(self, codes, scales, k=None):
        """``k``: columns that count, where ``codes`` has zeros behind them (default: all)."""
        torch = _torch()
        if not (isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor) and codes.is_cuda and scales.is_cuda):
            raise TypeError("Int8Weight expects torch CUDA tensors")
        if codes.dtype != torch.int8 or codes.ndim != 2 or not codes.numel():
            raise ValueError("codes must be a non-empty int8 matrix")
        n, columns = codes.shape
        k = columns if k is None else int(k)
        if not 1 <= k <= columns:
            raise ValueError(f"k must be within 1..{columns}")
        if scales.dtype != torch.float32 or scales.shape != (n,) or scales.device != codes.device:
            raise ValueError(f"scales must be FP32 [{n}] on {codes.device}")
        if k > INT8_MAX_K:
            raise NotImplementedError(f"sums of more than {INT8_MAX_K} products do not fit 32 bits")
        if n > INT8_MAX_SIZE:
            raise NotImplementedError(f"at most {INT8_MAX_SIZE} channels")
        padded = -(-k // 16) * 16
        if padded != columns:
            wide = torch.zeros((n, padded), dtype=torch.int8, device=codes.device)
            wide[:, :k] = codes[:, :k]
            codes = wide
        elif not codes.is_contiguous() or codes.data_ptr() % 16:
            codes = codes.clone(memory_format=torch.contiguous_format)
        self.codes, self.scales, self.shape, self.device = codes, scales.contiguous(), (n, k), codes.device

    @classmethod
    def quantize(cls, dense):
        """From a dense ``[N, K]`` matrix (FP32 / FP16 / BF16 CUDA tensor)."""
        if dense.ndim != 2:
            raise ValueError("a weight is a matrix")
        codes, scales = quantize_int8_rows(dense)
        return cls(codes, scales, dense.shape[1])

    @classmethod
    def from_packed(cls, packed):
        """From a packed GGUF matrix on the device (any format that ``quantized_linear`` takes)."""
        if not isinstance(packed, DevicePackedGGUFWeight):
            raise TypeError("Expected a DevicePackedGGUFWeight")
        return cls.quantize(dequantize_device(packed.data, packed.shape[0], packed.shape[1], packed.quant_type))

    @property
    def nbytes(self):
        return self.codes.numel() + 4 * self.scales.numel()


def int8_matmul(codes, scales, weight, *, out_dtype=None):
    """``(codes * scales) @ weight.T`` -> ``[rows, N]`` (FP32 unless ``out_dtype`` says otherwise) for rows from
    ``quantize_int8_rows``: one quantisation can serve several projections."""
    return _matmul("b200q_int8_gemm", codes, scales, weight, out_dtype)


def _matmul(entry, codes, scales, weight, out_dtype):
    torch = _torch()
    if not isinstance(weight, Int8Weight):
        raise TypeError("Expected an Int8Weight")
    n, k = weight.shape
    padded = weight.codes.shape[1]
    if (codes.dtype != torch.int8 or codes.ndim != 2 or codes.shape[1] != padded or not codes.is_contiguous()
            or scales.dtype != torch.float32 or scales.shape != (codes.shape[0],) or not scales.is_contiguous()):
        raise ValueError(f"Input does not match the weight (expected int8 [rows, {padded}] codes and FP32 [rows] scales)")
    if codes.device != weight.device or scales.device != weight.device:
        raise ValueError(f"activations must be on {weight.device}")
    out = torch.empty((codes.shape[0], n), dtype=out_dtype or torch.float32, device=codes.device)
    ident = _dtype_id(out, "out_dtype")
    if codes.data_ptr() % 16:
        raise ValueError("codes must be 16-byte aligned")
    if codes.shape[0] > INT8_MAX_SIZE:
        raise NotImplementedError(f"at most {INT8_MAX_SIZE} rows")
    if codes.shape[0]:
        _launch(codes.device, entry, weight.codes.data_ptr(), padded, weight.scales.data_ptr(), n, k, codes.data_ptr(),
                padded, scales.data_ptr(), codes.shape[0], out.data_ptr(), ident)
    return out


def int8_linear(x, weight, *, out_dtype=None):
    """``quantized_linear`` in 8-bit integers: quantises ``x`` ``[..., K]`` per token, then ``int8_matmul``; the output has x's
    leading shape and, by default, x's type."""
    if type(weight) is Int8Weight:
        host = _lib.host()
        if host is not None:
            y = host.int8_linear(x, weight.codes, weight.scales, weight.shape[0], weight.shape[1], out_dtype)
            if y is not None:
                return y
    if not isinstance(weight, Int8Weight):
        raise TypeError("Expected an Int8Weight")
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"Input K={x.shape[-1]} does not match weight K={weight.shape[1]}")
    codes, scales = _quantize(x, 1)
    y = _matmul("b200q_int8_gemm_behind_quantize", codes, scales, weight, out_dtype or x.dtype)
    return y.reshape(x.shape[:-1] + (weight.shape[0],))
