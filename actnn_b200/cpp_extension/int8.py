"""Matrix products in 8-bit integers, with a scale for each token and each output channel.

Codes of a matrix are one int8 a value and one float32 scale a row: ``value = code * scale``, ``scale = max|row| / 127``.
Rows of codes start on 16 bytes: ``quantize_rows`` returns a ``[.., K]`` view of rows padded with zeros to a multiple of 16.
A row that holds a NaN or an infinity decodes to NaN, its neighbours stay as they are.

The reference computes its linear layers in the activation's type (actnn/actnn/ops.py:408-428) and has no counterpart."""
import ctypes

import torch

from .. import _lib
from ._checks import FLOAT_TYPES, check_cuda_values

MOST_K = 131072                # 127 * 127 * K stays below 2^31


def _check_codes(codes, scale, name):
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda or not isinstance(scale, torch.Tensor):
        raise RuntimeError("%s must be a CUDA tensor!" % name)
    if codes.dtype != torch.int8 or scale.dtype != torch.float32:
        raise RuntimeError("The type of %s is not correct! (int8 codes, float32 scales)" % name)
    if codes.dim() < 1 or scale.shape != codes.shape[:-1]:
        raise RuntimeError("The dimension of %s is not correct!" % name)
    if scale.device != codes.device:
        raise RuntimeError("codes and scales of %s are on different devices" % name)


def _rows(codes):
    """``codes`` as a matrix whose rows start on 16 bytes, and the bytes between them; copied only when they do not."""
    k = codes.shape[-1]
    if codes.dim() != 2:
        codes = codes.reshape(-1, k) if k else codes.reshape(codes.shape[:-1].numel(), 0)
    ld = codes.stride(0) if codes.shape[0] > 1 else (k + 15) // 16 * 16
    if codes.stride(1) != 1 and k > 1 or ld % 16 or ld < k or codes.data_ptr() % 16:
        ld = (k + 15) // 16 * 16
        padded = torch.zeros(codes.shape[0], ld, dtype=torch.int8, device=codes.device)
        padded[:, :k] = codes
        codes = padded[:, :k]
    return codes, ld


def quantize_rows(x):
    """``(codes, scale)``: int8 ``[.., K]`` (rows padded to a multiple of 16 in memory) and float32 ``[..]``."""
    check_cuda_values(x, "x")
    if x.dim() < 1:
        raise RuntimeError("The dimension of x is not correct!")
    lead, k = x.shape[:-1], x.shape[-1]
    rows = lead.numel()
    if x.dim() == 2 and (x.stride(1) == 1 or k == 1) and (rows <= 1 or x.stride(0) >= k):
        flat, ld_x = x, (x.stride(0) if rows > 1 else k)
    else:
        flat, ld_x = x.contiguous(), k
    ld = (k + 15) // 16 * 16
    codes = torch.empty(lead + (ld,), dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    if k == 0:
        scale.fill_(1.0)
    _lib.call("actnn_row_codes", x, flat.data_ptr(), codes.data_ptr(), scale.data_ptr(), rows, k, ld_x, ld,
              _lib.dtype_id(x.dtype), _lib.stream_of(x))
    return codes[..., :k], scale


def dequantize_rows(codes, scale, dtype=torch.bfloat16):
    """``codes * scale`` in ``dtype``, contiguous."""
    _check_codes(codes, scale, "codes")
    flat, ld = _rows(codes)
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    _lib.call("actnn_row_decode", out, flat.data_ptr(), scale.contiguous().data_ptr(), out.data_ptr(), flat.shape[0],
              flat.shape[1], ld, _lib.dtype_id(dtype), _lib.stream_of(out))
    return out


def matmul(codes, scale, weight_codes, weight_scale, bias=None, dtype=torch.bfloat16):
    """``(codes * scale) @ (weight_codes * weight_scale).T + bias`` in ``dtype``: ``[.., K]`` by ``[N, K]`` gives ``[.., N]``."""
    _check_codes(codes, scale, "codes")
    _check_codes(weight_codes, weight_scale, "weight_codes")
    _check_product(codes, weight_codes, bias, dtype)
    flat, ld = _rows(codes)
    weights, ld_w = _rows(weight_codes)
    n, k = weights.shape
    out = torch.empty(codes.shape[:-1] + (n,), dtype=dtype, device=codes.device)
    if bias is not None:
        bias = bias.to(dtype).contiguous()
    if k == 0:                               # a sum of nothing
        return out.copy_(bias) if bias is not None else out.zero_()
    scale, weight_scale = scale.contiguous(), weight_scale.contiguous()
    _lib.call("actnn_int8_matmul", out, flat.data_ptr(), scale.data_ptr(), weights.data_ptr(), weight_scale.data_ptr(),
              _lib.ptr(bias), out.data_ptr(), flat.shape[0], n, k, ld, ld_w, _lib.dtype_id(dtype), _lib.stream_of(out))
    return out


def column_sums(x):
    """The sums over the rows of a matrix, in float32 and rounded once: the gradient of a bias."""
    check_cuda_values(x, "x")
    if x.dim() != 2:
        raise RuntimeError("The dimension of x is not correct!")
    x = x.contiguous()
    size = ctypes.c_int64(0)
    _lib.call("actnn_column_sums_workspace", x, x.shape[0], x.shape[1], ctypes.addressof(size))
    ws = _lib.scratch(x.device, size.value)
    out = torch.empty(x.shape[1], dtype=x.dtype, device=x.device)
    _lib.call("actnn_column_sums", x, x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], _lib.dtype_id(x.dtype), ws.data_ptr(),
              size.value, _lib.stream_of(x))
    return out


def _check_product(x, weight_codes, bias, dtype):
    if dtype not in FLOAT_TYPES:
        raise RuntimeError("actnn_b200: unsupported dtype %s" % dtype)
    if weight_codes.dim() != 2 or x.dim() < 1 or weight_codes.shape[1] != x.shape[-1]:
        raise RuntimeError("shapes %s and %s cannot be multiplied" % (tuple(x.shape), tuple(weight_codes.shape)))
    if x.shape[-1] > MOST_K:
        raise RuntimeError("a product over %d values may overflow its 32-bit sum; at most %d are accepted" % (x.shape[-1], MOST_K))
    if weight_codes.device != x.device:
        raise RuntimeError("the weight is on %s, the tokens on %s" % (weight_codes.device, x.device))
    if bias is not None:
        check_cuda_values(bias, "bias", x.device)
        if bias.dim() != 1 or bias.shape[0] != weight_codes.shape[0]:
            raise RuntimeError("The dimension of bias is not correct!")


def linear(x, weight_codes, weight_scale, bias=None):
    """A linear layer on a weight kept as codes: the tokens ``x`` ``[.., K]`` are coded row by row, the result has their type.
    No gradient passes through it: training goes through ``ops.int8_linear``."""
    nat = _lib.native()
    if nat:
        return nat.int8_linear(x, weight_codes, weight_scale, bias)
    check_cuda_values(x, "x")
    _check_codes(weight_codes, weight_scale, "weight_codes")
    _check_product(x, weight_codes, bias, x.dtype)
    codes, scale = quantize_rows(x)
    return matmul(codes, scale, weight_codes, weight_scale, bias, x.dtype)
