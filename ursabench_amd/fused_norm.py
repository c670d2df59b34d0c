"""Layer norm and the residual sum in front of it as gfx950 launches (K16, include/ursa_hip.h): what `fused_bn` is to the
convolutional blocks, for networks that normalise each row by itself.

`layer_norm(ln, x)` stands for `ln(x)`; `add_layer_norm(ln, (a, b))` for `z = a + b; return z, ln(z)`. `ln` stays a plain
`nn.LayerNorm` (state_dict keys, eps, no weight or no bias included); only the launches differ:

  forward           one launch: sum, statistics, scale and shift (and the 8-bit copy of z with `save8`)
  backward          one launch for dx (the gradient that reaches z past the norm added in it) and the columns' partial sums, and a
                    small one that adds those in a fixed order

float32, bfloat16 and float16 on a HIP device, parameters of the same type or float32, any width. Inputs that are not contiguous are
copied first. Anything else - host tensors, other types, autocast, empty tensors, a class or an instance with a forward of its own,
hooks on `ln` or on all modules, tensor subclasses, `torch.func` transforms, forward-mode derivatives, dispatch modes and tracing -
takes `ln(x)`, the stock path, where `save8` keeps the input itself. Double backward raises, and so do batched (`is_grads_batched`) and
dual gradients in the backward pass. On a HIP tensor the fused path needs csrc/libursa_hip.so and csrc/_ursa_torch.so, its autograd
nodes (no silent fallback: a missing library raises).

`save8=True` keeps the normalised input in 8 bits for the backward pass (K17, `act8`): gradients are the formula's with xhat
taken from those values; mean and 1 / std are the exact input's. `URSA_FUSED_NORM=0` / `enabled(False)` selects the stock path
everywhere (A/B runs).
"""
import math
import os

import torch
import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from . import _native

_TENSORS = frozenset((torch.Tensor, nn.Parameter, type(None)))       # a subclass may have a meaning of its own for every operator
_on = os.environ.get('URSA_FUSED_NORM', '1') != '0'


def enabled(flag=None):
    """Query / set the process-wide switch; returns the previous value."""
    global _on
    old = _on
    if flag is not None:
        _on = bool(flag)
    return old


def _fusable(ln, w, b, x):
    t, dev, shape = x.dtype, x.get_device(), ln.normalized_shape
    return (_on and x.is_cuda and t in _native.DTYPES and x.numel() > 0 and not torch.is_autocast_enabled()
            and type(ln).forward is nn.LayerNorm.forward and 'forward' not in ln.__dict__ and not _has_any_global_hook()
            and not (ln._forward_hooks or ln._forward_pre_hooks or ln._backward_hooks or ln._backward_pre_hooks)
            and type(x) in _TENSORS and type(w) in _TENSORS and type(b) in _TENSORS and x.shape[-len(shape):] == shape and ln.eps >= 0
            and (w is None or (w.get_device() == dev and (w.dtype is t or w.dtype is torch.float32)))
            and (b is None or (b.get_device() == dev and (b.dtype is t or b.dtype is torch.float32) and (w is None or w.dtype is b.dtype))))


def _flat(p):
    return p if p is None or (p.dim() == 1 and p.is_contiguous()) else p.reshape(-1).contiguous()


def _params(ln):
    own = ln._parameters                                  # (a parametrised weight is a property instead)
    return own['weight'] if 'weight' in own else ln.weight, own['bias'] if 'bias' in own else ln.bias


def layer_norm(ln, x, *, save8=False):
    """ln(x). save8: keep x in 8 bits for the backward pass (module docstring)."""
    if not isinstance(ln, nn.LayerNorm):
        raise TypeError(f'layer_norm wants an nn.LayerNorm, got {type(ln).__name__}')
    w, b = _params(ln)
    y = None
    if _fusable(ln, w, b, x):
        y = _native.nodes().layer_norm(x, _flat(w), _flat(b), math.prod(ln.normalized_shape), ln.eps, save8)
    return ln(x) if y is None else y                      # (None from there: the operands are more than memory to torch)


def add_layer_norm(ln, x, *, save8=False):
    """(z, ln(z)) for z = a + b of the pair x = (a, b); of a tensor x: (x, ln(x)). z is rounded to the tensors' type before it is
    normalised, as the two stock ops would do."""
    if not isinstance(x, tuple):
        return x, layer_norm(ln, x, save8=save8)
    if not isinstance(ln, nn.LayerNorm):
        raise TypeError(f'add_layer_norm wants an nn.LayerNorm, got {type(ln).__name__}')
    a, b = x
    w, bias = _params(ln)
    if _fusable(ln, w, bias, a) and b.shape == a.shape and b.dtype is a.dtype and b.device == a.device and type(b) in _TENSORS:
        pair = _native.nodes().add_layer_norm(a, b, _flat(w), _flat(bias), math.prod(ln.normalized_shape), ln.eps, save8)
        if pair is not None:
            return pair
    z = a + b
    return z, layer_norm(ln, z, save8=save8)
