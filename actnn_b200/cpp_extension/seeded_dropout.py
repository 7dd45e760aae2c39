"""Dropout from a counter-based generator whose mask is never stored: the backward pass draws it again.

A mask is a key ``(seed, offset)``: element i of the flattened tensor has the 16-bit field i % 8 of the Philox4x32-10 output for
counter i / 8, and is kept where field + 1 > 65536 p.  These are the fields of ``act_quantized_dropout``, which stores a bit for each
element: for one key the two give the same result.

The reference keeps a bit an element (actnn/actnn/cpp_extension/quantization.cc:128-148)."""
import torch

from .. import _lib
from ._checks import check_cuda_values, on_16_bytes

MASK64 = 0xFFFFFFFFFFFFFFFF


def check_probability(p):
    """``p`` as a float; at least 0 and below 1."""
    if not isinstance(p, (int, float)) or not 0 <= p < 1:
        raise RuntimeError("the dropout probability must be at least 0 and below 1, got %r" % (p,))
    return float(p)


def check_key(key):
    """``(seed, offset)`` as two 64-bit numbers."""
    if not isinstance(key, (tuple, list)) or len(key) != 2 or not all(isinstance(v, int) for v in key):
        raise RuntimeError("a key is a pair of whole numbers (seed, offset), got %r" % (key,))
    return key[0] & MASK64, key[1] & MASK64


def apply_mask(x, p, key, state=None):
    """``x`` with the elements that the key drops zeroed and the others divided by ``1 - p``; its own gradient is the same call.
    ``state``: an int64 tensor (seed, offset) on the device that is read in place of ``key``."""
    check_cuda_values(x, "x")
    p, (seed, offset) = check_probability(p), check_key(key)
    if state is not None and (state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous() or state.device != x.device):
        raise RuntimeError("state must be two int64 on the device of x")
    x = on_16_bytes(x)
    y = torch.empty_like(x)
    _lib.call("actnn_seeded_dropout", x, x.data_ptr(), y.data_ptr(), x.numel(), p, _lib.dtype_id(x.dtype), seed, offset,
              _lib.ptr(state), _lib.stream_of(x))
    return y
