"""Layer norm over the last dimension with a learned scale and shift.

    mean = mean_n x        var = mean_n (x - mean)^2
    xn   = (x - mean) / sqrt(var + eps)
    y    = xn * weight + bias

Stands beside `modnorm` (instance norm over the pixels of a channel with
a scale and shift per element) as the normalization of a TOKEN over its
channels. The HIP kernels (csrc/layer_norm.hip) run forward and first-order
backward, the sums over the rows for the parameters' gradients included;
a create_graph backward goes through the differentiable composition.
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


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = native.require_ext().layer_norm_fwd(
            x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.eps = eps
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        if torch.is_grad_enabled():
            # create_graph: differentiate the composition again, from the
            # inputs (the saved statistics are constants to autograd)
            return _eager_grads(
                lambda *t: _eager_layer_norm(*t, ctx.eps),
                (x, weight, bias), need, dy) + (None,)
        dx, dw, db = native.require_ext().layer_norm_bwd(
            dy, x, weight, bias, mean, rstd, need[0], need[1], need[2])
        return dx, dw, db, None


def _eager_grads(fn, inputs, need, dy):
    """Differentiable gradients of fn(*inputs) in those that need one.

    Through a view of each input: one input may come from another (a
    residual and the normalized residual), and the gradient of this
    operator alone must not run on into that history.
    """
    views = [None if t is None else t.view_as(t) for t in inputs]
    got = iter(torch.autograd.grad(
        fn(*views), [t for t, n in zip(views, need) if n], dy,
        create_graph=True))
    return tuple(next(got) if n else None for n in need[:len(inputs)])


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


_GPU_DTYPES = (torch.float32, torch.bfloat16)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Normalize x [..., N] over its last dimension.

    weight, bias: [N] in x's dtype or float32 (both in the same one), or
    None for a scale of 1 and a shift of 0. Returns x's shape and dtype;
    the statistics are held in 32 bits. On the GPU x is float32 or
    bfloat16. Rows may be strided (a slice of a wider tensor is read in
    place as long as its last dimension is contiguous).
    """
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x needs a last dimension of at "
                         f"least 1, got shape {tuple(x.shape)}")
    shape = (x.shape[-1],)
    _check_param("layer_norm: weight", weight, x, shape)
    _check_param("layer_norm: bias", bias, x, shape)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight is {weight.dtype}, "
                         f"bias {bias.dtype}")
    if not native.use_native(x):
        return _eager_layer_norm(x, weight, bias, eps)
    if x.dtype not in _GPU_DTYPES:
        raise ValueError(f"layer_norm: expected float32 or bfloat16 on the "
                         f"GPU, got {x.dtype}")
    if torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return native.require_ext().layer_norm_fwd(x, weight, bias, eps,
                                               False)[0]
