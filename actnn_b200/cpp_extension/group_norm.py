"""Group norm with an activation on channels-last tensors, its input kept in 8 bits for the backward pass.

Tensors are ``[N, C, ...]`` as ``nn.GroupNorm`` takes them.  The kernels read positions of consecutive channels: a
channels-last tensor is taken where it is, another one is copied; results are channels-last.  The codes of a (sample, group)
are 127 steps either way of the middle of its range.

The reference's norms are batch norms (actnn/actnn/ops.py:444-500); it has no counterpart of this one."""
import ctypes

import torch

from .. import _lib
from ._checks import activation_kind, activation_name, check_cuda_values


def _positions(x, name, groups):
    """``x`` as contiguous ``[N, ..., C]``, and N, S, C."""
    check_cuda_values(x, name)
    if x.dim() < 2:
        raise RuntimeError("The dimension of %s is not correct!" % name)
    n, c = x.shape[0], x.shape[1]
    if not isinstance(groups, int) or groups < 1 or c < 1 or c % groups:
        raise RuntimeError("%d channels cannot be split into %r groups" % (c, groups))
    last = x.movedim(1, -1).contiguous()
    return last, n, x.shape[2:].numel(), c


def _parameter(p, name, c, device):
    if p is None:
        return None
    check_cuda_values(p, name, device)
    if p.shape != (c,):
        raise RuntimeError("%s must have one value for each of the %d channels" % (name, c))
    return p.detach().float().contiguous()


def _workspace(x, n, s, c, groups):
    size = ctypes.c_int64(0)
    _lib.call("actnn_group_norm_workspace", x, n, s, c, groups, ctypes.addressof(size))
    return _lib.scratch(x.device, size.value), size.value


def _run(x, groups, weight, bias, eps, activation, codes_wanted, stats_wanted):
    kind = activation_kind(activation)
    last, n, s, c = _positions(x, "x", groups)
    weight, bias = _parameter(weight, "weight", c, x.device), _parameter(bias, "bias", c, x.device)
    y = torch.empty_like(last)
    codes = torch.empty(last.shape, dtype=torch.int8, device=x.device) if codes_wanted else None
    stats = torch.empty(n, groups, 4, dtype=torch.float32, device=x.device) if stats_wanted else None
    ws, size = _workspace(last, n, s, c, groups)
    _lib.call("actnn_group_norm_forward", last, last.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(), _lib.ptr(codes),
              _lib.ptr(stats), n, s, c, groups, float(eps), kind, _lib.dtype_id(x.dtype), ws.data_ptr(), size, _lib.stream_of(last))
    return y.movedim(-1, 1), last, codes, stats


def inference(x, groups, weight=None, bias=None, eps=1e-5, activation="none"):
    """The output alone."""
    nat = _lib.native()
    if nat:
        return nat.group_norm_value(x, groups, weight, bias, eps, activation_name(activation))
    return _run(x, groups, weight, bias, eps, activation, False, False)[0]


def forward(x, groups, weight=None, bias=None, eps=1e-5, activation="none", compress=True):
    """``(y, saved, stats)``: ``saved`` are the codes ``[N, ..., C]``, or with ``compress`` false the input itself in that order."""
    y, last, codes, stats = _run(x, groups, weight, bias, eps, activation, compress, True)
    return y, (codes if compress else last), stats


def backward(grad_y, saved, stats, groups, weight=None, bias=None, activation="none", parameter_grads=(True, True)):
    """``(grad_x, grad_weight, grad_bias)``; the latter float32, ``None`` where not asked for."""
    kind = activation_kind(activation)
    last, n, s, c = _positions(grad_y, "grad_y", groups)
    if saved.shape != last.shape or not saved.is_contiguous() or saved.device != last.device \
            or saved.dtype not in (torch.int8, last.dtype):
        raise RuntimeError("saved is not what forward returned for a gradient of this shape and type")
    if stats.shape != (n, groups, 4) or stats.dtype != torch.float32 or not stats.is_contiguous() or stats.device != last.device:
        raise RuntimeError("stats is not what forward returned for a gradient of this shape")
    weight, bias = _parameter(weight, "weight", c, last.device), _parameter(bias, "bias", c, last.device)
    grad_x = torch.empty_like(last)
    gw, gb = (torch.empty(c, dtype=torch.float32, device=last.device) if want else None for want in parameter_grads)
    coded = saved.dtype == torch.int8
    ws, size = _workspace(last, n, s, c, groups)
    _lib.call("actnn_group_norm_backward", last, last.data_ptr(), _lib.ptr(None if coded else saved),
              _lib.ptr(saved if coded else None), stats.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), grad_x.data_ptr(),
              _lib.ptr(gw), _lib.ptr(gb), n, s, c, groups, kind, _lib.dtype_id(last.dtype), ws.data_ptr(), size,
              _lib.stream_of(last))
    return grad_x.movedim(-1, 1), gw, gb
