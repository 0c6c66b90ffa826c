"""Layer norm over the last dimension with a learned scale and shift.

    mean = mean_n x        var = mean_n (x - mean)^2
    xn   = (x - mean) / sqrt(var + eps)
    y    = xn * weight + bias

Stands beside `modnorm` (instance norm over the pixels of a channel with
a scale and shift per element) as the normalization of a TOKEN over its
channels. The HIP kernels (csrc/layer_norm.hip) run forward and first-order
backward, the sums over the rows for the parameters' gradients included;
their autograd function (csrc/ext_rows.hip) sends a create_graph backward
through a differentiable composition, and so goes a call with forward-mode
tangents or under torch.jit.trace.
"""

from __future__ import annotations

import torch

from . import native


def _eager_layer_norm(x, weight, bias, eps):
    ft = torch.float64 if x.dtype == torch.float64 else torch.float32
    xf = x.to(ft)
    xc = xf - xf.mean(dim=-1, keepdim=True)
    y = xc * (xc.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    if weight is not None:
        y = y * weight.to(ft)
    if bias is not None:
        y = y + bias.to(ft)
    return y.to(x.dtype)


def _check_param(name, p, x, shape):
    if p is None:
        return
    if tuple(p.shape) != shape:
        raise ValueError(f"{name}: expected shape {shape}, "
                         f"got {tuple(p.shape)}")
    if p.device != x.device:
        raise ValueError(f"{name} is on {p.device}, x on {x.device}")
    if p.dtype != x.dtype and p.dtype != torch.float32:
        raise ValueError(f"{name}: expected {x.dtype} or torch.float32, "
                         f"got {p.dtype}")


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Normalize x [..., N] over its last dimension.

    weight, bias: [N] in x's dtype or float32 (both in the same one), or
    None for a scale of 1 and a shift of 0. Returns x's shape and dtype;
    the statistics are held in 32 bits. On the GPU x is float32 or
    bfloat16 and N below 2^30. Rows may be strided (a slice of a wider
    tensor is read in place as long as its last dimension is contiguous).
    """
    if x.is_cuda:  # checks its arguments likewise
        return native.require_ext().layer_norm(x, weight, bias, eps)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x needs a last dimension of at "
                         f"least 1, got shape {tuple(x.shape)}")
    shape = (x.shape[-1],)
    _check_param("layer_norm: weight", weight, x, shape)
    _check_param("layer_norm: bias", bias, x, shape)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight is {weight.dtype}, "
                         f"bias {bias.dtype}")
    return _eager_layer_norm(x, weight, bias, eps)
