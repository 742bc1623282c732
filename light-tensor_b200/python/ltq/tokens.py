"""Quantise / dequantise with parameters per row ("token"), on device tensors, through the C ABI."""
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
    rows, cols = x.shape
    pitch, step = x.stride()
    if step != 1 and cols > 1:
        raise ValueError("the elements of a row must be contiguous")
    if rows <= 1:
        return cols
    if pitch < cols:
        raise ValueError("the rows of a tensor must not overlap")
    return pitch


def check_qparams(qparams, rows, device_index):
    if not (qparams.dtype is torch.uint8 and qparams.get_device() == device_index >= 0 and qparams.numel() == 8 * rows and qparams.is_contiguous()):
        raise ValueError(f"parameters must be a contiguous uint8 CUDA tensor [{rows}, 8] on device {device_index}: one QParams per row")


# The current stream of a device as an integer.  (torch.cuda.current_stream builds an object for it, two microseconds: as long
# as the smallest of these kernels runs.)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def raw_stream(device_index):
    return _raw_stream(device_index)


def quantize_tokens(x, q=None, qparams=None, sums=None):
    """GetMinMax, ComputeQuantizationParams and Quantize of every row of x on its own.  x: float32 / float16 / bfloat16 CUDA
    [M, K], rows may be strided.  Returns (codes uint8 [M, K], parameters uint8 [M, 8] laid out as QParams, code sums
    int32 [M]); existing tensors may be passed in for them.  A row with an infinity or NaN gets scale NaN and codes 0.
    K at most 8421504, so that a sum of codes fits."""
    dev = x.get_device()
    if dev < 0 or x.dim() != 2:
        raise ValueError("ltq operates on CUDA tensors only (there is no CPU path): a matrix [tokens, features] is expected")
    M, K = x.shape
    code, ld = dtype_code(x.dtype), row_stride(x)
    if q is None:
        q = x.new_empty(M, K, dtype=torch.uint8)
    elif not (q.get_device() == dev and q.dtype is torch.uint8 and q.is_contiguous() and q.shape == x.shape):
        raise ValueError(f"q must be a contiguous uint8 CUDA tensor [{M}, {K}]")
    if qparams is None:
        qparams = x.new_empty(M, 8, dtype=torch.uint8)
    else:
        check_qparams(qparams, M, dev)
    if sums is None:
        sums = x.new_empty(M, dtype=torch.int32)
    elif not (sums.get_device() == dev and sums.dtype is torch.int32 and sums.is_contiguous() and sums.numel() == M):
        raise ValueError("sums must be a contiguous int32 CUDA tensor with one value per token")
    if M:
        check(lib().ltq_quantize_tokens_u8(x.data_ptr(), code, M, K, ld, q.data_ptr(), qparams.data_ptr(), sums.data_ptr(), dev, _raw_stream(dev)))
    return q, qparams, sums


def dequantize_tokens(q, qparams, dtype=torch.float32, out=None):
    """scale * (code - zero point) of every row: q uint8 CUDA [M, K] contiguous, qparams uint8 [M, 8].  Returns [M, K] of `dtype`
    (`out` if given; its rows may be strided)."""
    dev = q.get_device()
    if not (dev >= 0 and q.dtype is torch.uint8 and q.dim() == 2 and q.is_contiguous()):
        raise ValueError("codes must be a contiguous uint8 CUDA tensor [tokens, features] (there is no CPU path)")
    M, K = q.shape
    check_qparams(qparams, M, dev)
    code = dtype_code(dtype)
    if out is None:
        out, ld = q.new_empty(M, K, dtype=dtype), K
    elif not (out.get_device() == dev and out.dtype is dtype and out.shape == q.shape):
        raise ValueError(f"out must be a CUDA tensor [{M}, {K}] of {dtype}")
    else:
        ld = row_stride(out)
    if M:
        check(lib().ltq_dequantize_tokens_u8(out.data_ptr(), code, ld, q.data_ptr(), qparams.data_ptr(), M, K, dev, _raw_stream(dev)))
    return out
