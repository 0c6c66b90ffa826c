"""Matrix product with bias, activation and residual in its epilogue.

    z = weight_gain * x @ weight^T + bias_gain * bias
    y = clamp(act(z) * gain) + residual

One kernel where `linear_nobias` and `bias_act` take a scaled copy of the
weight, a library product, a bias/activation pass and an addition. Backward:

    dz = dy * gain * act'(z), zero where |gain * act(z)| >= clamp
    dx = weight_gain * dz @ weight      dweight = weight_gain * dz^T @ x
    dbias = bias_gain * sum_rows dz     dresidual = dy

Sums, z and dz are held in 32 bits (a bf16 dz enters its two products as two
bf16 numbers), and every result is rounded once. All products run on the kernels
of csrc/linear_act.hip. A backward that needs z takes it from the product
again, or from 32 bits kept by the forward where that is quicker. The autograd
function (csrc/ext_rows.hip) sends a create_graph backward through a
differentiable composition, and so goes a call with forward-mode tangents or
under torch.jit.trace.
"""

from __future__ import annotations

import math

import torch

from . import native
from .fused_act import _eager_act, activation_defs
from .layer_norm import _check_param

# bias_act's activations and the two smooth ones of feed-forward layers:
# gelu(z) = z * Phi(z) (exact, by erf) and silu(z) = z * sigmoid(z)
linear_activations = {
    **activation_defs,
    "gelu": (5, 0.0, 1.0, True),
    "silu": (6, 0.0, 1.0, True),
}


def _act(z, act, alpha):
    if act == "gelu":
        return z * 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return _eager_act(z, act, alpha)


def _eager_linear_act(x, weight, bias, residual, act, alpha, gain, clamp,
                      weight_gain, bias_gain):
    ft = torch.float64 if x.dtype == torch.float64 else torch.float32
    z = x.to(ft).matmul(weight.to(ft).t()) * weight_gain
    if bias is not None:
        z = z + bias.to(ft) * bias_gain
    y = _act(z, act, alpha) * gain
    if clamp is not None:
        # clamp's own gradient would pass where y just reaches it; the
        # kernels' and bias_act's is 0 there
        y = torch.where(y.abs() >= clamp, y.detach().clamp(-clamp, clamp), y)
    if residual is not None:
        y = y + residual.to(ft)
    return y.to(x.dtype)


def linear_act(x, weight, bias=None, act="linear", residual=None, alpha=None,
               gain=None, clamp=None, weight_gain=1.0, bias_gain=1.0):
    """clamp(act(weight_gain * x @ weight^T + bias_gain * bias) * gain)
    + residual.

    x: [..., K]; weight: [N, K] in x's dtype; bias: [N] in x's dtype or
    float32; residual: [..., N] in x's dtype, added after the clamp. act is
    one of `linear_activations`, with `bias_act`'s default alpha and gain.
    clamp: None or negative for none. Returns [..., N] in x's dtype, rounded
    once from 32 bits. On the GPU x is float32 or bfloat16, the weight below
    2^20 a side and the rows of x fewer than 2^30; x, weight and residual may
    have strided rows, and rows that repeat or overlap (for the gradients of
    a weight those of x and of the incoming gradient are then copied).
    """
    spec = linear_activations.get(act)
    if spec is None:
        raise ValueError(f"linear_act: unknown activation {act!r}")
    if alpha is None:
        alpha = spec[1]
    if gain is None:
        gain = spec[2]
    if clamp is not None and clamp < 0:
        clamp = None
    if x.is_cuda:  # checks its arguments likewise
        return native.require_ext().linear_act(
            x, weight, bias, residual, spec[0], alpha, gain,
            math.inf if clamp is None else clamp, weight_gain, bias_gain)
    if x.ndim < 1 or weight.ndim != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"linear_act: x {tuple(x.shape)} and weight "
                         f"{tuple(weight.shape)} do not fit")
    n, k = weight.shape
    if n < 1 or k < 1:
        raise ValueError(f"linear_act: empty weight {tuple(weight.shape)}")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError(f"linear_act: weight is {weight.dtype} on "
                         f"{weight.device}, x {x.dtype} on {x.device}")
    _check_param("linear_act: bias", bias, x, (n,))
    if residual is not None:
        if residual.shape != x.shape[:-1] + (n,):
            raise ValueError(f"linear_act: residual {tuple(residual.shape)} "
                             f"does not fit the output "
                             f"{tuple(x.shape[:-1]) + (n,)}")
        if residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"linear_act: residual is {residual.dtype} on "
                             f"{residual.device}, x {x.dtype} on {x.device}")
    return _eager_linear_act(x, weight, bias, residual, act, alpha, gain,
                             clamp, weight_gain, bias_gain)
