"""Layer norm and the residual sum in front of it as gfx950 launches (K16, include/ursa_hip.h): what `fused_bn` is to the
convolutional blocks, for networks that normalise each row by itself.

`layer_norm(ln, x)` stands for `ln(x)`; `add_layer_norm(ln, (a, b))` for `z = a + b; return z, ln(z)`. `ln` stays a plain
`nn.LayerNorm` (state_dict keys, eps, no weight or no bias included); only the launches differ:

  forward           one launch: sum, statistics, scale and shift (and the 8-bit copy of z with `save8`)
  backward          one launch for dx (the gradient that reaches z past the norm added in it) and the columns' partial sums, and a
                    small one that adds those in a fixed order

float32, bfloat16 and float16 on a HIP device, parameters of the same type or float32, any width. Inputs that are not contiguous are
copied first. Anything else - host tensors, other types, autocast, empty tensors, a subclass with a forward of its own, hooks on
`ln` - takes `ln(x)`, the stock path, where `save8` keeps the input itself. Double backward is not offered. On a HIP tensor the
fused path needs csrc/libursa_hip.so (no silent fallback: a missing library raises).

`save8=True` keeps the normalised input in 8 bits for the backward pass (K17, `act8`): gradients are the formula's with xhat
taken from those values; mean and 1 / std are the exact input's. `URSA_FUSED_NORM=0` / `enabled(False)` selects the stock path
everywhere (A/B runs).
"""
import math
import os

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native

_on = os.environ.get('URSA_FUSED_NORM', '1') != '0'


def enabled(flag=None):
    """Query / set the process-wide switch; returns the previous value."""
    global _on
    old = _on
    if flag is not None:
        _on = bool(flag)
    return old


def _gradients(ctx, dy, dz, need_x, need_w, need_b):
    z, q, e, stats, w = ctx.saved_tensors
    return _native.default_kernels().layer_norm_backward(
        dy.contiguous(), stats, w, x=z, q=q, e=e, dz=None if dz is None else dz.contiguous(), need_dx=need_x,
        param_type=ctx.param_type, need_dgamma=need_w, need_dbeta=need_b)


class _Norm(torch.autograd.Function):
    """y = layer_norm(x) for 2-d contiguous x."""

    @staticmethod
    def forward(ctx, x, w, b, eps, save8):
        z, y, ms, q, e = _native.default_kernels().layer_norm(x, w, b, eps=eps, stats=True, save8=save8)
        ctx.save_for_backward(None if save8 else z, q, e, ms, w)
        ctx.param_type = None if b is None else b.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*_gradients(ctx, dy, None, *ctx.needs_input_grad[:3]), None, None)


class _AddNorm(torch.autograd.Function):
    """(z, y) = (a + b, layer_norm(a + b)); d(a) = d(b) = dz + the norm's gradient, in the same launch."""

    @staticmethod
    def forward(ctx, a, b, w, bias, eps, save8):
        ctx.set_materialize_grads(False)                 # an unused output's gradient arrives as None, not as zeros
        z, y, ms, q, e = _native.default_kernels().layer_norm(a, w, bias, eps=eps, addend=b, stats=True, save8=save8)
        ctx.save_for_backward(None if save8 else z, q, e, ms, w)
        ctx.param_type = None if bias is None else bias.dtype
        return z, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dz, dy):
        need_a, need_b, need_w, need_bias = ctx.needs_input_grad[:4]
        if dy is None:                                   # y unused: only the sum's own gradient flows
            return dz if need_a else None, dz if need_b else None, None, None, None, None
        dx, dw, db = _gradients(ctx, dy, dz, need_a or need_b, need_w, need_bias)
        return dx if need_a else None, dx if need_b else None, dw, db, None, None


def _fusable(ln, w, b, x):
    t, dev, shape = x.dtype, x.get_device(), ln.normalized_shape
    return (_on and x.is_cuda and t in _native.DTYPES and x.numel() > 0 and not torch.is_autocast_enabled()
            and type(ln).forward is nn.LayerNorm.forward
            and not (ln._forward_hooks or ln._forward_pre_hooks or ln._backward_hooks or ln._backward_pre_hooks)
            and x.shape[-len(shape):] == shape and ln.eps >= 0
            and (w is None or (w.get_device() == dev and (w.dtype is t or w.dtype is torch.float32)))
            and (b is None or (b.get_device() == dev and (b.dtype is t or b.dtype is torch.float32) and (w is None or w.dtype is b.dtype))))


def _rows(n, x):
    """x as rows of its last n dimensions."""
    if n == 1:
        return (x if x.dim() == 2 else x.reshape(-1, x.shape[-1])).contiguous()
    return x.flatten(x.dim() - n).reshape(-1, math.prod(x.shape[x.dim() - n:])).contiguous()


def _flat(p):
    return p if p is None or (p.dim() == 1 and p.is_contiguous()) else p.reshape(-1).contiguous()


def _params(ln):
    own = ln._parameters                                  # (a parametrised weight is a property instead)
    return own['weight'] if 'weight' in own else ln.weight, own['bias'] if 'bias' in own else ln.bias


def _recorded(x, w, b, addend=None):
    return torch.is_grad_enabled() and (x.requires_grad or (w is not None and w.requires_grad) or (b is not None and b.requires_grad)
                                        or (addend is not None and addend.requires_grad))


def layer_norm(ln, x, *, save8=False):
    """ln(x). save8: keep x in 8 bits for the backward pass (module docstring)."""
    if not isinstance(ln, nn.LayerNorm):
        raise TypeError(f'layer_norm wants an nn.LayerNorm, got {type(ln).__name__}')
    w, b = _params(ln)
    if not _fusable(ln, w, b, x):
        return ln(x)
    n = len(ln.normalized_shape)
    flat = n == 1 and x.dim() == 2
    x2, w, b = _rows(n, x), _flat(w), _flat(b)
    if _recorded(x, w, b):
        y = _Norm.apply(x2, w, b, ln.eps, save8)
    else:
        y = _native.default_kernels().layer_norm(x2, w, b, eps=ln.eps)[1]
    return y if flat else y.view(x.shape)


def add_layer_norm(ln, x, *, save8=False):
    """(z, ln(z)) for z = a + b of the pair x = (a, b); of a tensor x: (x, ln(x)). z is rounded to the tensors' type before it is
    normalised, as the two stock ops would do."""
    if not isinstance(x, tuple):
        return x, layer_norm(ln, x, save8=save8)
    if not isinstance(ln, nn.LayerNorm):
        raise TypeError(f'add_layer_norm wants an nn.LayerNorm, got {type(ln).__name__}')
    a, b = x
    w, bias = _params(ln)
    if not (_fusable(ln, w, bias, a) and b.shape == a.shape and b.dtype is a.dtype and b.device == a.device):
        z = a + b
        return z, layer_norm(ln, z, save8=save8)
    n = len(ln.normalized_shape)
    flat = n == 1 and a.dim() == 2
    a2, b2, w, bias = _rows(n, a), _rows(n, b), _flat(w), _flat(bias)
    if _recorded(a, w, bias, b):
        z, y = _AddNorm.apply(a2, b2, w, bias, ln.eps, save8)
    else:
        z, y = _native.default_kernels().layer_norm(a2, w, bias, eps=ln.eps, addend=b2)[:2]
    return (z, y) if flat else (z.view(a.shape), y.view(a.shape))
