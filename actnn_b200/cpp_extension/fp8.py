"""Matrix products in 8-bit floating point (e4m3) with a power-of-two scale for each block of 128.

Of a block, e is the least integer, at least -126, with max|block| <= 448 * 2^e; a code is x * 2^-e rounded to e4m3 and stands for
code * 2^e.  Blocks are 128 consecutive values of a row (``quantize``), or squares of 128 x 128 (``quantize_weight``).  Codes are
``torch.float8_e4m3fn``, rows on 16 bytes.  Scales are bytes e + 127, in the order in which the tensor cores read them: uint8
``[ceil(K / 512), ceil(rows / 128), 512]``, of 128 rows and four blocks that of row r and block j at (r % 32) * 16 + (r / 32) * 4 + j.
A value that is not finite is coded as NaN; its neighbours stay as they are.

The reference computes its linear layers in the activation's type (actnn/actnn/ops.py:408-428) and has no counterpart."""
import ctypes

import torch

from .. import _lib
from ._checks import FLOAT_TYPES, check_cuda_values

BLOCK = 128
CODES = torch.float8_e4m3fn


def _row_bytes(k):
    return (k + 15) // 16 * 16


def _scale_shape(rows, k):
    return ((k + 511) // 512, (rows + 127) // 128, 512)


def _check_codes(codes, scales, name):
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda or not isinstance(scales, torch.Tensor):
        raise RuntimeError("%s must be a CUDA tensor!" % name)
    if codes.dtype != CODES or scales.dtype != torch.uint8:
        raise RuntimeError("The type of %s is not correct! (float8_e4m3fn codes, uint8 scales)" % name)
    if codes.dim() < 1 or tuple(scales.shape) != _scale_shape(codes.shape[:-1].numel(), codes.shape[-1]):
        raise RuntimeError("The dimension of %s is not correct!" % name)
    if scales.device != codes.device:
        raise RuntimeError("codes and scales of %s are on different devices" % name)


def _rows(codes):
    """``codes`` as a matrix of bytes whose rows start on 16 bytes, and the bytes between them; copied only when they do not."""
    k = codes.shape[-1]
    codes = codes.view(torch.uint8)
    if codes.dim() != 2:
        codes = codes.reshape(codes.shape[:-1].numel(), k)
    ld = codes.stride(0) if codes.shape[0] > 1 else _row_bytes(k)
    if codes.stride(1) != 1 and k > 1 or ld % 16 or ld < k or codes.data_ptr() % 16:
        ld = _row_bytes(k)
        padded = torch.zeros(codes.shape[0], ld, dtype=torch.uint8, device=codes.device)
        padded[:, :k] = codes
        codes = padded[:, :k]
    return codes, ld


def _on_16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _matrix(x):
    """``x`` as a matrix of evenly spaced rows, and the elements between them; copied only where they are not."""
    check_cuda_values(x, "x")
    if x.dim() < 1:
        raise RuntimeError("The dimension of x is not correct!")
    rows, k = x.shape[:-1].numel(), x.shape[-1]
    if x.dim() == 2 and (x.stride(1) == 1 or k == 1) and (rows <= 1 or x.stride(0) >= k):
        return x, rows, k, (x.stride(0) if rows > 1 else k)
    return x.contiguous(), rows, k, k


def _empty(rows, k, device):
    return torch.empty(rows, _row_bytes(k), dtype=torch.uint8, device=device), torch.empty(_scale_shape(rows, k), dtype=torch.uint8, device=device)


def quantize(x):
    """``(codes, scales)`` of ``[.., K]`` in blocks of 128 values of a row."""
    flat, rows, k, ld = _matrix(x)
    codes, scales = _empty(rows, k, x.device)
    _lib.call("actnn_fp8_row_codes", x, flat.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, k, ld, codes.shape[1],
              _lib.dtype_id(x.dtype), _lib.stream_of(x))
    return codes.view(CODES).view(x.shape[:-1] + codes.shape[1:])[..., :k], scales


def quantize_weight(weight, both=False):
    """``(codes, scales)`` of a matrix in squares of 128 x 128; with ``both`` also those of its transpose, which stand for the same."""
    if weight.dim() != 2:
        raise RuntimeError("The dimension of weight is not correct!")
    rowwise, transposed, _ = tile_codes(weight, True, both, False, square=True)
    return rowwise + transposed if both else rowwise


def tile_codes(x, rowwise=True, transposed=True, sums=False, square=False):
    """``((codes, scales), (codes, scales) of the transpose, column sums of 128 rows each)`` of a matrix read once, ``None`` what is not
    asked for.  The transpose is coded in blocks of 128 rows of ``x``."""
    flat, rows, k, ld = _matrix(x)
    here, there = _empty(rows, k, x.device) if rowwise else None, _empty(k, rows, x.device) if transposed else None
    parts = torch.empty((rows + 127) // 128, k, dtype=torch.float32, device=x.device) if sums else None
    if rowwise or transposed or sums:
        (c, s), (ct, st) = here or (None, None), there or (None, None)
        _lib.call("actnn_fp8_tile_codes", x, flat.data_ptr(), _lib.ptr(c), _lib.ptr(s), _lib.ptr(ct), _lib.ptr(st), _lib.ptr(parts), rows, k, ld,
                  _row_bytes(k), _row_bytes(rows), int(square), _lib.dtype_id(x.dtype), _lib.stream_of(x))
    def view(pair, n):
        return None if pair is None else (pair[0].view(CODES)[:, :n], pair[1])
    return view(here, k), view(there, rows), parts


def join_sums(parts, dtype):
    """The sums over the rows of ``parts``, in float32 and rounded once."""
    out = torch.empty(parts.shape[1], dtype=dtype, device=parts.device)
    _lib.call("actnn_fp8_join_sums", out, parts.data_ptr(), out.data_ptr(), parts.shape[0], parts.shape[1], _lib.dtype_id(dtype),
              _lib.stream_of(out))
    return out


def dequantize(codes, scales, dtype=torch.bfloat16):
    """What the codes stand for, in ``dtype``, contiguous."""
    _check_codes(codes, scales, "codes")
    flat, ld = _rows(codes)
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    _lib.call("actnn_fp8_decode", out, flat.data_ptr(), _on_16(scales).data_ptr(), out.data_ptr(), flat.shape[0], flat.shape[1], ld,
              _lib.dtype_id(dtype), _lib.stream_of(out))
    return out


def _check_product(x, weight_codes, bias, dtype):
    if dtype not in FLOAT_TYPES:
        raise RuntimeError("actnn_b200: unsupported dtype %s" % dtype)
    if weight_codes.dim() != 2 or x.dim() < 1 or weight_codes.shape[1] != x.shape[-1]:
        raise RuntimeError("shapes %s and %s cannot be multiplied" % (tuple(x.shape), tuple(weight_codes.shape)))
    if weight_codes.device != x.device:
        raise RuntimeError("the weight is on %s, the tokens on %s" % (weight_codes.device, x.device))
    if bias is not None:
        check_cuda_values(bias, "bias", x.device)
        if bias.dim() != 1 or bias.shape[0] != weight_codes.shape[0]:
            raise RuntimeError("The dimension of bias is not correct!")


def matmul(codes, scales, weight_codes, weight_scales, bias=None, dtype=torch.bfloat16):
    """The product of what the codes stand for, plus ``bias``, in ``dtype``: ``[.., K]`` by ``[N, K]`` gives ``[.., N]``."""
    _check_codes(codes, scales, "codes")
    _check_codes(weight_codes, weight_scales, "weight_codes")
    _check_product(codes, weight_codes, bias, dtype)
    flat, ld = _rows(codes)
    weights, ld_w = _rows(weight_codes)
    n, k = weights.shape
    out = torch.empty(codes.shape[:-1] + (n,), dtype=dtype, device=codes.device)
    if bias is not None:
        bias = bias.detach().to(dtype).contiguous()
    if k == 0:                               # a sum of nothing
        return out.copy_(bias) if bias is not None else out.zero_()
    scales, weight_scales = _on_16(scales), _on_16(weight_scales)
    _lib.call("actnn_fp8_matmul", out, flat.data_ptr(), scales.data_ptr(), weights.data_ptr(), weight_scales.data_ptr(), _lib.ptr(bias),
              out.data_ptr(), flat.shape[0], n, k, ld, ld_w, _lib.dtype_id(dtype), _lib.stream_of(out))
    return out


def linear(x, weight_codes, weight_scales, bias=None):
    """A linear layer on a weight kept as codes: the tokens ``x`` ``[.., K]`` are coded row by row, the result has their type.
    No gradient passes through it: training goes through ``ops.fp8_linear``."""
    nat = _lib.native()
    if nat:
        return nat.fp8_linear(x, weight_codes, weight_scales, bias)
    check_cuda_values(x, "x")
    _check_codes(weight_codes, weight_scales, "weight_codes")
    _check_product(x, weight_codes, bias, x.dtype)
    flat, rows, k, ld = _matrix(x)
    weights, ld_w = _rows(weight_codes)
    out = torch.empty(x.shape[:-1] + weights.shape[:1], dtype=x.dtype, device=x.device)
    if bias is not None:
        bias = bias.detach().to(x.dtype).contiguous()
    if k == 0:
        return out.copy_(bias) if bias is not None else out.zero_()
    size = ctypes.c_int64(0)
    _lib.call("actnn_fp8_linear_workspace", x, rows, k, ctypes.addressof(size))
    ws = _lib.scratch(x.device, size.value) if size.value else None
    weight_scales = _on_16(weight_scales)
    _lib.call("actnn_fp8_linear", x, flat.data_ptr(), weights.data_ptr(), weight_scales.data_ptr(), _lib.ptr(bias), out.data_ptr(), rows,
              weights.shape[0], k, ld, ld_w, _lib.dtype_id(x.dtype), _lib.ptr(ws), size.value, _lib.stream_of(x))
    return out
