"""Activation functions whose backward pass reads an 8-bit copy of the input instead of the input.

``activation``: "none", "relu", "silu", "gelu" (erf) or "gelu_tanh".  The gated form takes ``[.., 2 * F]`` and gives
``f(x[.., :F]) * x[.., F:]``.  256 consecutive elements (of each half) share a float32 scale, their largest magnitude over 127.

Of the reference's activation functions only ReLU saves less than its input (one bit,
actnn/actnn/cpp_extension/quantization.cc:106-124); it has no counterpart of these."""
import torch

from .. import _lib
from ._checks import activation_kind, check_cuda_values, on_16_bytes

BLOCK = 256


def activation_forward(x, activation, gated=False, save=True):
    """``(y, codes, scale)``; codes and scale are ``None`` unless ``save``."""
    kind = activation_kind(activation)
    check_cuda_values(x, "x")
    cols = x.shape[-1] if x.dim() else 1
    if gated:
        if x.dim() < 1 or cols % 2:
            raise RuntimeError("a gated activation splits its last dimension in two, got shape %s" % (tuple(x.shape),))
        cols //= 2
    x = on_16_bytes(x)
    shape = x.shape[:-1] + (cols,) if x.dim() else x.shape
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    numel = y.numel()
    codes = scale = None
    if save:
        blocks = (numel + BLOCK - 1) // BLOCK * (2 if gated else 1)
        codes = torch.empty(blocks * BLOCK, dtype=torch.int8, device=x.device)
        scale = torch.empty(blocks, dtype=torch.float32, device=x.device)
    if numel:
        _lib.call("actnn_act_forward", x, x.data_ptr(), y.data_ptr(), _lib.ptr(codes), _lib.ptr(scale), numel // cols, cols,
                  int(gated), kind, _lib.dtype_id(x.dtype), _lib.stream_of(x))
    return y, codes, scale


def activation_backward(grad_y, activation, codes=None, scale=None, x=None, gated=False):
    """The gradient of the input, from the codes of the forward pass or (``codes`` None) from the input ``x`` itself."""
    kind = activation_kind(activation)
    check_cuda_values(grad_y, "grad_y")
    grad_y = on_16_bytes(grad_y)
    numel, cols = grad_y.numel(), grad_y.shape[-1] if grad_y.dim() else 1
    shape = grad_y.shape[:-1] + (2 * cols,) if gated else grad_y.shape
    blocks = (numel + BLOCK - 1) // BLOCK * (2 if gated else 1)
    if codes is not None:
        if codes.dtype != torch.int8 or scale is None or scale.dtype != torch.float32:
            raise RuntimeError("The type of codes is not correct!")
        if codes.numel() != blocks * BLOCK or scale.numel() != blocks or not codes.is_contiguous() or not scale.is_contiguous():
            raise RuntimeError("codes and scale are not those of an activation with %d outputs" % numel)
        if codes.device != grad_y.device or scale.device != grad_y.device:
            raise RuntimeError("codes and grad_y are on different devices")
    else:
        check_cuda_values(x, "x", grad_y.device)
        if x.shape != shape or x.dtype != grad_y.dtype:
            raise RuntimeError("x must have the shape %s and the type of grad_y" % (tuple(shape),))
        x = on_16_bytes(x)
    grad_x = torch.empty(shape, dtype=grad_y.dtype, device=grad_y.device)
    if numel:
        _lib.call("actnn_act_backward", grad_y, grad_y.data_ptr(), _lib.ptr(x if codes is None else None), _lib.ptr(codes),
                  _lib.ptr(scale), grad_x.data_ptr(), numel // cols, cols, int(gated), kind, _lib.dtype_id(grad_y.dtype),
                  _lib.stream_of(grad_y))
    return grad_x
