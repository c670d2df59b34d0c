"""The linear layer with its epilogue, act(x W' + b) + residual, as gfx950 launches (K15, include/ursa_hip.h).

`linear_act(fc, x, activation, residual)` stands for `F.relu(self.fc1(x))` and the like (URSABench/models/mlp.py:20-23) and for the
`out += residual` behind it. `fc` stays a plain `nn.Linear` (same state_dict keys, initialisation and optimizer view); only the
launches differ:

  forward           one launch: product, bias, activation and residual (two where the contraction is cut over workgroups)
  backward          the activation's gradient and the bias gradient in one pass over dy, then dx and dW by the same product kernel

float32, bfloat16 and float16, any sizes and leading dimensions, on a HIP device. Operands that are not contiguous are copied first.
Anything else - host tensors, other or mixed types, autocast, a class or an instance with a forward of its own, hooks on `fc` or on
all modules, tensor subclasses, `torch.func` transforms, forward-mode derivatives, dispatch modes and tracing - takes `fc(x)`, the
activation and the sum as stock ops, where `save8` keeps x itself. Double backward raises, and so do batched (`is_grads_batched`) and
dual gradients in the backward pass. On a HIP tensor the fused path needs csrc/libursa_hip.so and csrc/_ursa_torch.so, its autograd
nodes (no silent fallback: a missing library raises).

`save8=True` keeps the x that the weight gradient needs in 8 bits (K17, `act8`) instead of the tensor: a quarter / half of its
memory, dW as if x had been rounded to 8 bits per block of 32 features; y, dx and db do not change.

In a captured step take gradients with `torch.autograd.grad`, or drop every eager graph of the same parameters before the capture:
their accumulation nodes are bound to the stream of the first graph that uses them, whichever operator that is.

`URSA_FUSED_LINEAR=0` / `enabled(False)` selects the stock ops in `linear_act` everywhere (A/B runs). `URSA_LINEAR_IN_MODELS=1` /
`in_models(True)` makes `models.MLP` and `models.LeNet5` call it (off by default: their products stay the library's, bit for bit).
"""
import os

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook

from . import _native

_on = os.environ.get('URSA_FUSED_LINEAR', '1') != '0'
_models = os.environ.get('URSA_LINEAR_IN_MODELS', '0') == '1'
_TENSORS = frozenset((torch.Tensor, nn.Parameter, type(None)))       # a subclass may have a meaning of its own for every operator
_STOCK = {None: lambda z: z, 'relu': F.relu, 'gelu': F.gelu, 'silu': F.silu}


def enabled(flag=None):
    """Query / set whether `linear_act` takes this module's launches at all (process-wide); returns the previous value."""
    global _on
    old = _on
    if flag is not None:
        _on = bool(flag)
    return old


def in_models(flag=None):
    """Query / set whether models.MLP / models.LeNet5 run their linear layers through `linear_act` (process-wide)."""
    global _models
    old = _models
    if flag is not None:
        _models = bool(flag)
    return old


def _fusable(fc, w, b, x, residual):
    t, dev = x.dtype, x.get_device()
    return (_on and x.is_cuda and t in _native.DTYPES and x.dim() >= 1 and not torch.is_autocast_enabled()
            and type(fc).forward is nn.Linear.forward and 'forward' not in fc.__dict__ and not _has_any_global_hook()
            and not (fc._forward_hooks or fc._forward_pre_hooks or fc._backward_hooks or fc._backward_pre_hooks)
            and type(x) in _TENSORS and type(w) in _TENSORS and type(b) in _TENSORS and type(residual) in _TENSORS
            and w.dtype is t and w.get_device() == dev and x.shape[-1] == w.shape[1] and w.numel() > 0
            and (b is None or (b.dtype is t and b.get_device() == dev))
            and (residual is None or (residual.dtype is t and residual.get_device() == dev)))


def linear_act(fc, x, activation=None, residual=None, *, save8=False):
    """act(fc(x)) + residual. activation: None, 'relu', 'gelu' (the exact one, z Phi(z)) or 'silu'; residual: None or a tensor of
    the result's shape. save8: keep x in 8 bits for the weight gradient (module docstring)."""
    if activation not in _STOCK:
        raise ValueError(f'activation must be one of {list(_STOCK)}, got {activation!r}')
    if not isinstance(fc, nn.Linear):
        raise TypeError(f'linear_act wants an nn.Linear, got {type(fc).__name__}')
    own = fc._parameters                                  # (a parametrised weight is a property instead)
    w = own['weight'] if 'weight' in own else fc.weight
    b = own['bias'] if 'bias' in own else fc.bias
    shape = x.shape[:-1] + (w.shape[0],)
    if residual is not None and residual.shape != shape:
        raise ValueError(f'residual {tuple(residual.shape)} should have the result\'s shape {tuple(shape)}')
    if _fusable(fc, w, b, x, residual):
        y = _native.nodes().linear_act(x, w, b, residual, _native.ACTIVATIONS[activation], save8)
        if y is not None:                                 # (None: the operands are more than memory to torch)
            return y
    y = _STOCK[activation](fc(x))
    return y if residual is None else y + residual
