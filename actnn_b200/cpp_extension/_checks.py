"""Argument checks with the reference's error texts (ext_common.h:2-27)."""
import torch

FLOAT_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def check_cuda_tensor(t, name, ndim=None, dtype=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError("%s must be a CUDA tensor!" % name)
    if not t.is_contiguous():
        raise RuntimeError("%s must be contiguous!" % name)
    if ndim is not None and t.dim() != ndim:
        raise RuntimeError("The dimension of %s is not correct!" % name)
    if dtype is None:
        if t.dtype not in FLOAT_TYPES:
            raise RuntimeError("The type of %s is not correct!" % name)
    elif t.dtype != dtype:
        raise RuntimeError("The type of %s is not correct!" % name)


ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def activation_kind(name):
    """The library's number of an activation function (``None`` counts as "none")."""
    try:
        return ACTIVATIONS["none" if name is None else name]
    except (KeyError, TypeError):
        raise RuntimeError("activation must be one of %s, got %r" % (", ".join(sorted(ACTIVATIONS)), name)) from None


def activation_name(name):
    """The name that both halves of the binding take for what a caller named, or ``None``."""
    activation_kind(name)
    return "none" if name is None else name


def check_cuda_values(t, name, device=None):
    """A floating CUDA tensor of a supported type, any strides; on ``device`` when given."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError("%s must be a CUDA tensor!" % name)
    if t.dtype not in FLOAT_TYPES:
        raise RuntimeError("The type of %s is not correct!" % name)
    if device is not None and t.device != device:
        raise RuntimeError("%s is on %s, expected %s" % (name, t.device, device))


def on_16_bytes(t):
    """``t`` contiguous with its data on 16 bytes; copied only when it is not."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
