"""The norms before and after a block with its gate and residual scale, in one pass:

    r = scale * x + gate * drop(norm(branch) * post_weight + post_bias)        h = norm(r) * weight + bias

``x`` is the residual stream, ``branch`` the block's output, ``h`` what the next block reads.  ``kind``: "rms" (without biases) or
"layer"; ``post`` false leaves the first norm out.  Parameters are ``[C]`` or ``None``; a gate has the last dimension C and before it the leading
dimensions of ``x`` up to some place, ones behind it (``[C]``, ``[B, 1, C]``, ``[B, S, C]``).

For the backward pass ``x`` and ``branch`` are kept in 8 bits: 256 consecutive channels of a row share a float32 scale, their largest
magnitude over 127.  The mask of the dropout is not kept (``seeded_dropout``).

The reference's norms are batch norms (actnn/actnn/ops.py:444-500); it has no counterpart of this one."""
import ctypes

import torch
from torch.autograd import forward_ad

from .. import _lib
from ._checks import FLOAT_TYPES, check_cuda_values
from .seeded_dropout import check_key, check_probability

MOST_CHANNELS = 32768
KINDS = {"rms": 0, "layer": 1}
CHANNELS = 256                 # that share a scale


def norm_kind(kind):
    try:
        return KINDS[kind]
    except (KeyError, TypeError):
        raise RuntimeError("kind must be one of layer, rms, got %r" % (kind,)) from None


def _no_tangents(**tensors):
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("%s has a forward-mode tangent, which residual_norm does not pass on" % name)


def _inputs(x, branch):
    check_cuda_values(x, "x")
    check_cuda_values(branch, "branch", x.device)
    if x.dim() < 1 or branch.shape != x.shape:
        raise RuntimeError("x and branch must have the same shape of at least one dimension, got %s and %s" % (tuple(x.shape), tuple(branch.shape)))
    if not 1 <= x.shape[-1] <= MOST_CHANNELS:
        raise RuntimeError("a row has %d channels; 1 to %d are accepted" % (x.shape[-1], MOST_CHANNELS))
    if x.shape[:-1].numel() > 0x7fffffff:
        raise RuntimeError("%d rows are more than 2^31 - 1" % x.shape[:-1].numel())


def _parameters(x, weight, bias, post_weight, post_bias, post, layer):
    """The four as contiguous tensors of one type, and that type."""
    given = {"weight": weight, "bias": bias, "post_weight": post_weight, "post_bias": post_bias}
    for name, p in given.items():
        if p is None:
            continue
        if not layer and name.endswith("bias"):
            raise RuntimeError("%s belongs to the kind \"layer\"" % name)
        if not post and name.startswith("post"):
            raise RuntimeError("%s without the norm that it belongs to" % name)
        check_cuda_values(p, name, x.device)
        if p.shape != x.shape[-1:]:
            raise RuntimeError("%s must have one value for each of the %d channels" % (name, x.shape[-1]))
    types = {p.dtype for p in given.values() if p is not None}
    dtype = types.pop() if len(types) == 1 else torch.float32
    return tuple(None if p is None else p.detach().to(dtype).contiguous() for p in given.values()), dtype


def gate_rows(x, gate):
    """How many rows of ``x`` share a row of ``gate``."""
    if gate is None:
        return max(1, x.shape[:-1].numel())
    check_cuda_values(gate, "gate", x.device)
    lead, own = x.shape[:-1], gate.shape[:-1]
    own = (1,) * (len(lead) - len(own)) + tuple(own)
    j = 0
    while j < len(lead) and len(own) == len(lead) and own[j] == lead[j]:
        j += 1
    if gate.dim() < 1 or gate.shape[-1] != x.shape[-1] or len(own) != len(lead) or any(n != 1 for n in own[j:]):
        raise RuntimeError("a gate of shape %s does not belong to rows of shape %s: it has the channels and before them the leading "
                           "dimensions up to some place" % (tuple(gate.shape), tuple(x.shape)))
    return max(1, lead[j:].numel())


def run(x, branch, weight=None, bias=None, post_weight=None, post_bias=None, gate=None, scale=1.0, p=0.0, eps=1e-5, kind="rms", post=True,
        key=(0, 0), codes=False, stats=False):
    """``(r, h, codes, stats)``: ``codes`` is ``(codes of x, their scales, codes of branch, their scales)`` or ``None``, ``stats`` the
    rows' means and reciprocal deviations, two of each."""
    layer, p, (seed, offset) = norm_kind(kind), check_probability(p), check_key(key)
    _inputs(x, branch)
    if branch.dtype != x.dtype:
        raise RuntimeError("x and branch must have the same type")
    _no_tangents(x=x, branch=branch, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate)
    params, pdtype = _parameters(x, weight, bias, post_weight, post_bias, post, layer)
    each = gate_rows(x, gate)
    gate = None if gate is None else gate.detach().contiguous()
    x, branch = x.contiguous(), branch.contiguous()
    c, rows = x.shape[-1], x.shape[:-1].numel()
    r, h = torch.empty_like(x), torch.empty_like(x)
    kept = None
    if codes:
        blocks = (c + CHANNELS - 1) // CHANNELS
        kept = tuple(torch.empty(s, dtype=t, device=x.device) for _ in range(2) for s, t in (((rows, c), torch.int8), ((rows, blocks), torch.float32)))
    st = torch.empty(rows, 4, dtype=torch.float32, device=x.device) if stats or codes else None
    cx, sx, cf, sf = kept or (None,) * 4
    _lib.call("actnn_residual_norm_forward", x, x.data_ptr(), branch.data_ptr(), *(_lib.ptr(q) for q in params), _lib.ptr(gate), r.data_ptr(),
              h.data_ptr(), _lib.ptr(cx), _lib.ptr(cf), _lib.ptr(sx), _lib.ptr(sf), _lib.ptr(st), rows, c, each, float(scale), float(eps),
              layer, int(bool(post)), p, _lib.dtype_id(x.dtype), _lib.dtype_id(pdtype),
              _lib.dtype_id(x.dtype if gate is None else gate.dtype), seed, offset, None, _lib.stream_of(x))
    return r, h, kept, st


def inference(x, branch, weight=None, bias=None, post_weight=None, post_bias=None, gate=None, scale=1.0, eps=1e-5, kind="rms", post=True):
    """``(r, h)`` alone, without dropout.  No gradient passes through it: training goes through ``ops.residual_norm``."""
    nat = _lib.native()
    if nat:
        return nat.residual_norm_value(x, branch, weight, bias, post_weight, post_bias, gate, float(scale), 0.0, float(eps), norm_kind(kind),
                                       bool(post), None)
    return run(x, branch, weight, bias, post_weight, post_bias, gate, scale, 0.0, eps, kind, post)[:2]


def backward(grad_r, grad_h, saved, stats, weight=None, bias=None, post_weight=None, post_bias=None, gate=None, scale=1.0, p=0.0, kind="rms",
             post=True, key=(0, 0), wanted=(True,) * 7):
    """The gradients of x, branch, weight, bias, post_weight, post_bias and gate, ``None`` where not wanted.  ``saved``: what ``run``
    returned as codes, or ``(x, branch)``.  One of the two gradients may be ``None``."""
    layer, p, (seed, offset) = norm_kind(kind), check_probability(p), check_key(key)
    like = grad_r if grad_r is not None else grad_h
    if like is None:
        raise RuntimeError("one of grad_r and grad_h must be given")
    for g, name in ((grad_r, "grad_r"), (grad_h, "grad_h")):
        if g is not None:
            check_cuda_values(g, name, like.device)
            if g.shape != like.shape or g.dtype != like.dtype:
                raise RuntimeError("grad_r and grad_h must have the same shape and type")
    c, rows = like.shape[-1], like.shape[:-1].numel()
    params, pdtype = _parameters(like, weight, bias, post_weight, post_bias, post, layer)
    each = gate_rows(like, gate)
    flat = None if gate is None else gate.detach().contiguous()
    gdtype = like.dtype if gate is None else gate.dtype
    coded = len(saved) == 4
    cx, sx, cf, sf = saved if coded else (None,) * 4
    x, f = (None, None) if coded else saved
    for t, n, dtype in (((cx, rows * c, torch.int8), (cf, rows * c, torch.int8)) if coded else ((x, rows * c, like.dtype), (f, rows * c, like.dtype))) \
            + ((stats, rows * 4, torch.float32),):
        if t.numel() != n or t.dtype != dtype or not t.is_contiguous() or t.device != like.device:
            raise RuntimeError("saved and stats are not what the forward pass left for a gradient of this shape and type")
    grad_r, grad_h = (None if g is None else g.contiguous() for g in (grad_r, grad_h))
    gx, gf = (torch.empty(like.shape, dtype=like.dtype, device=like.device) if w else None for w in wanted[:2])
    grads = [torch.empty(c, dtype=pdtype, device=like.device) if w and q is not None else None for w, q in zip(wanted[2:6], params)]
    gg = torch.empty(gate.shape, dtype=gate.dtype, device=like.device) if gate is not None and wanted[6] else None
    if rows == 0:
        return (gx, gf) + tuple(None if g is None else g.zero_() for g in grads + [gg])
    size = ctypes.c_int64(0)
    _lib.call("actnn_residual_norm_workspace", like, rows, c, each, int(gg is not None), ctypes.addressof(size))
    ws = _lib.scratch(like.device, size.value)
    _lib.call("actnn_residual_norm_backward", like, _lib.ptr(grad_r), _lib.ptr(grad_h), _lib.ptr(x), _lib.ptr(f), _lib.ptr(cx), _lib.ptr(cf),
              _lib.ptr(sx), _lib.ptr(sf), stats.data_ptr(), _lib.ptr(params[0]), _lib.ptr(params[2]), _lib.ptr(params[3]), _lib.ptr(flat),
              _lib.ptr(gx), _lib.ptr(gf), *(_lib.ptr(g) for g in grads), _lib.ptr(gg), rows, c, each, float(scale), layer, int(bool(post)), p,
              _lib.dtype_id(like.dtype), _lib.dtype_id(pdtype), _lib.dtype_id(gdtype), seed, offset, None, ws.data_ptr(), size.value,
              _lib.stream_of(like))
    out = [None if g is None else g.to(q.dtype) for g, q in zip(grads, (weight, bias, post_weight, post_bias))]
    return (gx, gf) + tuple(out) + (gg,)
