"""Quantise / dequantise with parameters per row ("token"), on device tensors, through the C ABI."""
import ctypes as C

import torch

from ._binding import DTYPE_BF16, DTYPE_F16, DTYPE_F32, check, lib

_CODES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


def dtype_code(dtype):
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"float32, float16 or bfloat16 expected, not {dtype}")
    return code


def row_stride(x):
    """Elements between the rows of a 2-D tensor whose rows are contiguous."""
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError("the elements of a row must be contiguous")
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        raise ValueError("the rows of a tensor must not overlap")
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def check_qparams(qparams, rows, device_index):
    if not (qparams.is_cuda and qparams.dtype == torch.uint8 and qparams.is_contiguous() and qparams.numel() == 8 * rows
            and qparams.device.index == device_index):
        raise ValueError(f"parameters must be a contiguous uint8 CUDA tensor [{rows}, 8] on device {device_index}: one QParams per row")


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def quantize_tokens(x, q=None, qparams=None, sums=None):
    """GetMinMax, ComputeQuantizationParams and Quantize of every row of x on its own.  x: float32 / float16 / bfloat16 CUDA
    [M, K], rows may be strided.  Returns (codes uint8 [M, K], parameters uint8 [M, 8] laid out as QParams, code sums
    int32 [M]); existing tensors may be passed in for them.  A row with an infinity or NaN gets scale NaN and codes 0."""
    if not (x.is_cuda and x.dim() == 2):
        raise ValueError("ltq operates on CUDA tensors only (there is no CPU path): a matrix [tokens, features] is expected")
    M, K = x.shape
    code, ld = dtype_code(x.dtype), row_stride(x)
    if q is None:
        q = torch.empty((M, K), dtype=torch.uint8, device=x.device)
    elif not (q.device == x.device and q.dtype == torch.uint8 and q.is_contiguous() and q.shape == x.shape):
        raise ValueError(f"q must be a contiguous uint8 CUDA tensor [{M}, {K}]")
    if qparams is None:
        qparams = torch.empty((M, 8), dtype=torch.uint8, device=x.device)
    check_qparams(qparams, M, x.device.index)
    if sums is None:
        sums = torch.empty(M, dtype=torch.int32, device=x.device)
    elif not (sums.device == x.device and sums.dtype == torch.int32 and sums.is_contiguous() and sums.numel() == M):
        raise ValueError("sums must be a contiguous int32 CUDA tensor with one value per token")
    if M:
        check(lib().ltq_quantize_tokens_u8(x.data_ptr(), code, M, K, ld, q.data_ptr(), qparams.data_ptr(), sums.data_ptr(), x.device.index,
                                           _stream(x.device)))
    return q, qparams, sums


def dequantize_tokens(q, qparams, dtype=torch.float32, out=None):
    """scale * (code - zero point) of every row: q uint8 CUDA [M, K] contiguous, qparams uint8 [M, 8].  Returns [M, K] of `dtype`
    (`out` if given; its rows may be strided)."""
    if not (q.is_cuda and q.dtype == torch.uint8 and q.dim() == 2 and q.is_contiguous()):
        raise ValueError("codes must be a contiguous uint8 CUDA tensor [tokens, features] (there is no CPU path)")
    M, K = q.shape
    check_qparams(qparams, M, q.device.index)
    if out is None:
        out = torch.empty((M, K), dtype=dtype, device=q.device)
    elif not (out.device == q.device and out.dtype == dtype and out.shape == q.shape):
        raise ValueError(f"out must be a CUDA tensor [{M}, {K}] of {dtype}")
    code, ld = dtype_code(dtype), row_stride(out)
    if M:
        check(lib().ltq_dequantize_tokens_u8(out.data_ptr(), code, ld, q.data_ptr(), qparams.data_ptr(), M, K, q.device.index,
                                             _stream(q.device)))
    return out
