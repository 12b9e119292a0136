"""torch.library registration of the hot-path ops (SURVEY.md §8b "Wrappers").

The reference exposed its CUDA correlation through a cffi extension plus an autograd.Function
(correlation_package/functions/correlation.py:7-56, _ext/correlation/__init__.py:6-15), which
graph capture tools cannot see into.  Here each op is a ``torch.library.custom_op`` in the
``pwcnet`` namespace -- an opaque node with a fake (meta) implementation for shape
propagation and a registered autograd formula -- so ``torch.compile`` / FX / ``torch.export``
trace ``Correlation``, ``WarpingLayer`` and ``CostVolumeLayer`` as single nodes:

    torch.ops.pwcnet.correlation(in1, in2, pad, k, md, s1, s2, mult)   cu:34-106
    torch.ops.pwcnet.correlation_backward(in1, in2, gO, pad, ...)      cu:108-290
    torch.ops.pwcnet.cost_volume(src, tgt, sr) / _backward             modules.py:53-74
    torch.ops.pwcnet.warp(x, flow) / warp_backward                     modules.py:31-42
    torch.ops.pwcnet.layer_norm / rotary / linear / gated_linear       (features.py)

The real implementations are the HIP kernels behind the C ABI (ops.py); there is no CPU
kernel, so calling these ops on CPU tensors raises, as the reference's CPU stubs did.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import features as _features
from . import ops as _ops

_NS = "pwcnet"


def _on(t: Tensor):
    """The tensor's HIP device as current device (CPU tensors fall through to ops.py, which
    raises: there is no CPU implementation)."""
    import contextlib
    return torch.cuda.device(t.device) if t.is_cuda else contextlib.nullcontext()


def corr_output_shape(H: int, W: int, pad: int, k: int, md: int, s1: int, s2: int):
    """correlation_cuda.c:20-34 (C semantics: truncating integer division, float ceil)."""
    import math
    kr = int((k - 1) / 2)
    br = kr + md
    dr = md // s2
    D = 2 * dr + 1
    Ho = int(math.ceil((H + 2 * pad - 2 * br) / float(s1)))
    Wo = int(math.ceil((W + 2 * pad - 2 * br) / float(s1)))
    return D * D, max(Ho, 0), max(Wo, 0)


# ---------------------------------------------------------------------------------------
# correlation
# ---------------------------------------------------------------------------------------
@torch.library.custom_op(f"{_NS}::correlation", mutates_args=())
def correlation(input1: Tensor, input2: Tensor, pad_size: int, kernel_size: int,
                max_displacement: int, stride1: int, stride2: int,
                corr_multiply: int) -> Tensor:
    with _on(input1):
        return _ops.corr_forward(input1, input2, pad_size, kernel_size, max_displacement,
                                 stride1, stride2, corr_multiply)


@correlation.register_fake
def _(input1, input2, pad_size, kernel_size, max_displacement, stride1, stride2, corr_multiply):
    B, _, H, W = input1.shape
    OC, Ho, Wo = corr_output_shape(H, W, pad_size, kernel_size, max_displacement, stride1,
                                   stride2)
    return input1.new_empty((B, OC, Ho, Wo))


@torch.library.custom_op(f"{_NS}::correlation_backward", mutates_args=())
def correlation_backward(input1: Tensor, input2: Tensor, grad_output: Tensor, pad_size: int,
                         kernel_size: int, max_displacement: int, stride1: int, stride2: int,
                         corr_multiply: int) -> Tuple[Tensor, Tensor]:
    with _on(input1):
        return _ops.corr_backward(input1, input2, grad_output, pad_size, kernel_size,
                                  max_displacement, stride1, stride2, corr_multiply)


@correlation_backward.register_fake
def _(input1, input2, grad_output, *args):
    return torch.empty_like(input1), torch.empty_like(input2)


def _corr_setup(ctx, inputs, output):
    input1, input2, *params = inputs
    ctx.save_for_backward(input1, input2)
    ctx.params = params


def _corr_bwd(ctx, grad):
    input1, input2 = ctx.saved_tensors
    g1, g2 = correlation_backward(input1, input2, grad.contiguous(), *ctx.params)
    return (g1, g2) + (None,) * 6


correlation.register_autograd(_corr_bwd, setup_context=_corr_setup)


# ---------------------------------------------------------------------------------------
# CostVolumeLayer
# ---------------------------------------------------------------------------------------
@torch.library.custom_op(f"{_NS}::cost_volume", mutates_args=())
def cost_volume(src: Tensor, tgt: Tensor, search_range: int) -> Tensor:
    with _on(src):
        return _ops.cost_volume_forward(src, tgt, search_range)


@cost_volume.register_fake
def _(src, tgt, search_range):
    B, _, H, W = src.shape
    return src.new_empty((B, (2 * search_range + 1) ** 2, H, W))


@torch.library.custom_op(f"{_NS}::cost_volume_backward", mutates_args=())
def cost_volume_backward(src: Tensor, tgt: Tensor, grad_output: Tensor,
                         search_range: int) -> Tuple[Tensor, Tensor]:
    with _on(src):
        return _ops.cost_volume_backward(src, tgt, grad_output, search_range)


@cost_volume_backward.register_fake
def _(src, tgt, grad_output, search_range):
    return torch.empty_like(src), torch.empty_like(tgt)


def _cvl_setup(ctx, inputs, output):
    src, tgt, sr = inputs
    ctx.save_for_backward(src, tgt)
    ctx.sr = sr


def _cvl_bwd(ctx, grad):
    src, tgt = ctx.saved_tensors
    gs, gt = cost_volume_backward(src, tgt, grad.contiguous(), ctx.sr)
    return gs, gt, None


cost_volume.register_autograd(_cvl_bwd, setup_context=_cvl_setup)


# ---------------------------------------------------------------------------------------
# WarpingLayer
# ---------------------------------------------------------------------------------------
@torch.library.custom_op(f"{_NS}::warp", mutates_args=())
def warp(x: Tensor, flow: Tensor) -> Tensor:
    with _on(x):
        return _ops.warp_forward(x, flow)


@warp.register_fake
def _(x, flow):
    return torch.empty_like(x)


@torch.library.custom_op(f"{_NS}::warp_backward", mutates_args=())
def warp_backward(x: Tensor, flow: Tensor, grad_output: Tensor) -> Tuple[Tensor, Tensor]:
    with _on(x):
        return _ops.warp_backward(x, flow, grad_output)


@warp_backward.register_fake
def _(x, flow, grad_output):
    return torch.empty_like(x), torch.empty_like(flow)


def _warp_setup(ctx, inputs, output):
    x, flow = inputs
    ctx.save_for_backward(x, flow)


def _warp_bwd(ctx, grad):
    x, flow = ctx.saved_tensors
    gx, gf = warp_backward(x, flow, grad.contiguous())
    return gx, gf


warp.register_autograd(_warp_bwd, setup_context=_warp_setup)


# ---------------------------------------------------------------------------------------
# feature operators (features.py)
# ---------------------------------------------------------------------------------------
def _tokens(x, channel_dim):
    n = 1
    for d, size in enumerate(x.shape):
        if d != channel_dim % x.dim():
            n = n * size
    return n


@torch.library.custom_op(f"{_NS}::layer_norm", mutates_args=())
def layer_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
               channel_dim: int) -> Tuple[Tensor, Tensor, Tensor]:
    """(y, mean, rstd); mean and rstd have no gradient."""
    return _features.layer_norm_forward(x, weight, bias, eps, channel_dim, True)


@layer_norm.register_fake
def _(x, weight, bias, eps, channel_dim):
    n = _tokens(x, channel_dim)
    return (x.new_empty(x.shape), x.new_empty((n,), dtype=torch.float32),
            x.new_empty((n,), dtype=torch.float32))


@torch.library.custom_op(f"{_NS}::layer_norm_backward", mutates_args=())
def layer_norm_backward(x: Tensor, weight: Optional[Tensor], grad: Tensor, mean: Tensor,
                        rstd: Tensor, channel_dim: int) -> Tuple[Tensor, Tensor, Tensor]:
    return _features.layer_norm_backward(x, weight, grad, mean, rstd, channel_dim)


@layer_norm_backward.register_fake
def _(x, weight, grad, mean, rstd, channel_dim):
    C = x.shape[channel_dim]
    return x.new_empty(x.shape), x.new_empty((C,)), x.new_empty((C,))


def _norm_setup(ctx, inputs, output):
    x, weight, bias, eps, ctx.channel_dim = inputs
    ctx.has = (weight is not None, bias is not None)
    ctx.mark_non_differentiable(output[1], output[2])  # for the backward pass, and as they are
    ctx.save_for_backward(x, weight, output[1], output[2])


def _norm_bwd(ctx, grad, grad_mean, grad_rstd):
    x, weight, mean, rstd = ctx.saved_tensors
    gx, gw, gb = layer_norm_backward(x, weight, grad.contiguous(), mean, rstd, ctx.channel_dim)
    return gx, gw if ctx.has[0] else None, gb if ctx.has[1] else None, None, None


layer_norm.register_autograd(_norm_bwd, setup_context=_norm_setup)


@torch.library.custom_op(f"{_NS}::rotary", mutates_args=())
def rotary(x: Tensor, inv_freq: Tensor, axis: Tensor, positions: Optional[Tensor],
           grid: Optional[List[int]], origin: Optional[List[int]], interleaved: bool,
           inverse: bool) -> Tensor:
    return _features.rotary_forward(x, inv_freq, axis, positions, grid, origin, interleaved,
                                    inverse)


@rotary.register_fake
def _(x, inv_freq, axis, positions, grid, origin, interleaved, inverse):
    return torch.empty_like(x)


def _rotary_setup(ctx, inputs, output):
    x, inv_freq, axis, positions, *ctx.args = inputs
    if any(ctx.needs_input_grad[1:4]):
        raise ValueError("rotary: positions and inv_freq have no gradient")
    ctx.save_for_backward(inv_freq, axis, positions)


def _rotary_bwd(ctx, grad):
    inv_freq, axis, positions = ctx.saved_tensors
    grid, origin, interleaved, inverse = ctx.args
    g = rotary(grad, inv_freq, axis, positions, grid, origin, interleaved, not inverse)
    return (g,) + (None,) * 7


rotary.register_autograd(_rotary_bwd, setup_context=_rotary_setup)


def _product_fake(x, weight, channel_dim, halves):
    shape = list(x.shape)
    shape[channel_dim] = weight.shape[0] // halves
    return x.new_empty(shape)


@torch.library.custom_op(f"{_NS}::linear", mutates_args=())
def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor],
           activation: str, negative_slope: float, channel_dim: int) -> Tensor:
    return _features.linear_forward(x, weight, bias, residual, activation, negative_slope,
                                    channel_dim)


@linear.register_fake
def _(x, weight, bias, residual, activation, negative_slope, channel_dim):
    return _product_fake(x, weight, channel_dim, 1)


@torch.library.custom_op(f"{_NS}::linear_backward", mutates_args=())
def linear_backward(x: Tensor, weight: Tensor, bias: Optional[Tensor], grad: Tensor,
                    activation: str, negative_slope: float,
                    channel_dim: int) -> Tuple[Tensor, Tensor, Tensor]:
    return _features.linear_backward(x, weight, bias, grad, activation, negative_slope,
                                     channel_dim)


@torch.library.custom_op(f"{_NS}::gated_linear", mutates_args=())
def gated_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], activation: str,
                 negative_slope: float, channel_dim: int) -> Tensor:
    return _features.gated_linear_forward(x, weight, bias, activation, negative_slope,
                                          channel_dim)


@gated_linear.register_fake
def _(x, weight, bias, activation, negative_slope, channel_dim):
    return _product_fake(x, weight, channel_dim, 2)


@torch.library.custom_op(f"{_NS}::gated_linear_backward", mutates_args=())
def gated_linear_backward(x: Tensor, weight: Tensor, bias: Optional[Tensor], grad: Tensor,
                          activation: str, negative_slope: float,
                          channel_dim: int) -> Tuple[Tensor, Tensor, Tensor]:
    return _features.gated_linear_backward(x, weight, bias, grad, activation, negative_slope,
                                           channel_dim)


def _product_backward_fake(x, weight, *args):
    return (x.new_empty(x.shape), weight.new_empty(weight.shape),
            weight.new_empty((weight.shape[0],)))


linear_backward.register_fake(_product_backward_fake)
gated_linear_backward.register_fake(_product_backward_fake)


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, *ctx.args = inputs
    ctx.has = (bias is not None, residual is not None)
    ctx.save_for_backward(x, weight, bias)


def _linear_bwd(ctx, grad):
    x, weight, bias = ctx.saved_tensors
    gx, gw, gb = linear_backward(x, weight, bias, grad.contiguous(), *ctx.args)
    return (gx, gw, gb if ctx.has[0] else None, grad if ctx.has[1] else None, None, None, None)


def _gated_setup(ctx, inputs, output):
    x, weight, bias, *ctx.args = inputs
    ctx.has_bias = bias is not None
    ctx.save_for_backward(x, weight, bias)


def _gated_bwd(ctx, grad):
    x, weight, bias = ctx.saved_tensors
    gx, gw, gb = gated_linear_backward(x, weight, bias, grad.contiguous(), *ctx.args)
    return gx, gw, gb if ctx.has_bias else None, None, None, None


linear.register_autograd(_linear_bwd, setup_context=_linear_setup)
gated_linear.register_autograd(_gated_bwd, setup_context=_gated_setup)
