"""nn.Module drop-ins for the reference's hot-path layers.

* ``Correlation``     — correlation_package/modules/correlation.py:6-27 (same ctor, no params)
* ``WarpingLayer``    — modules.py:25-42 (ctor takes the reference's ``args`` namespace)
* ``CostVolumeLayer`` — modules.py:45-74 (ctor reads ``args.search_range``)
* ``WarpCorrelation`` — model.py:80-83 (warp, then correlation) as one module / one launch
* ``layer_norm``, ``rotary``, ``linear``, ``gated_linear`` and their modules ``LayerNorm``,
  ``RotaryPosition``, ``ChannelLinear``, ``GatedLinear``, ``FeatureBlock`` — the feature operators
  (features.py; no counterpart in the reference)
* ``get_grid``        — utils.py:3-8 (host-built normalised base grid, for API completeness;
  the HIP warp recomputes it in registers and never calls this)
"""
from __future__ import annotations

import math

import torch
from torch import nn

from . import features as _features
from . import library as _library  # registers torch.ops.pwcnet.* (traceable single nodes)
from .ops import (CorrelationCatFunction, UpsampleWarpFunction, WarpCorrelationFunction)


class Correlation(nn.Module):
    """``Correlation(pad_size, kernel_size, max_displacement, stride1, stride2, corr_multiply)``.

    ``forward(input1, input2)`` -> B x ((md/s2)*2+1)^2 x Ho x Wo, values of
    correlation_cuda_kernel.cu:34-106 (divided by kernel_size^2 * C).  model.py:24 builds it
    as Correlation(pad_size=9, kernel_size=1, max_displacement=9, stride1=1, stride2=2).
    """

    def __init__(self, pad_size=0, kernel_size=0, max_displacement=0, stride1=1, stride2=2,
                 corr_multiply=1):
        super().__init__()
        self.pad_size = pad_size
        self.kernel_size = kernel_size
        self.max_displacement = max_displacement
        self.stride1 = stride1
        self.stride2 = stride2
        self.corr_multiply = corr_multiply

    def forward(self, input1, input2):
        # functions/correlation.py:17-18 asserts contiguity; the op (torch.ops.pwcnet.
        # correlation, autograd registered) is CorrelationFunction's traceable twin
        assert input1.is_contiguous()
        assert input2.is_contiguous()
        return _library.correlation(input1, input2, self.pad_size, self.kernel_size,
                                    self.max_displacement, self.stride1, self.stride2,
                                    self.corr_multiply)

    def extra_repr(self):
        return (f"pad_size={self.pad_size}, kernel_size={self.kernel_size}, "
                f"max_displacement={self.max_displacement}, stride1={self.stride1}, "
                f"stride2={self.stride2}")


class WarpingLayer(nn.Module):
    """Backward-warp ``x`` by ``flow`` (pixels; channel 0 horizontal, 1 vertical).

    Matches modules.py:31-42 under the reference's pinned torch 0.4 (grid_sample bilinear,
    zeros padding, align_corners=True).  ``args`` is kept for signature parity; the device is
    taken from the inputs.
    """

    def __init__(self, args=None):
        super().__init__()
        self.args = args

    def forward(self, x, flow):
        return _library.warp(x, flow)


class WarpCorrelation(nn.Module):
    """One pyramid level of model.py:80-83 in one call:

        x2_warp = self.warping_layer(x2, flow)      # model.py:80
        corr = self.corr(x1, x2_warp)               # model.py:83
    becomes
        corr, x2_warp = self.warp_corr(x1, x2, flow)

    Same ctor as ``Correlation`` (model.py:24's values by default).  Values equal the two
    reference layers applied in sequence; gradients flow to x1, x2 and flow.
    """

    def __init__(self, pad_size=9, kernel_size=1, max_displacement=9, stride1=1, stride2=2,
                 corr_multiply=1):
        super().__init__()
        self.pad_size = pad_size
        self.kernel_size = kernel_size
        self.max_displacement = max_displacement
        self.stride1 = stride1
        self.stride2 = stride2
        self.corr_multiply = corr_multiply

    def forward(self, x1, x2, flow):
        return WarpCorrelationFunction.apply(x1, x2, flow, self.pad_size, self.kernel_size,
                                             self.max_displacement, self.stride1, self.stride2,
                                             self.corr_multiply)


class CorrelationCat(nn.Module):
    """model.py:83-91 in one call:

        corr = self.corr(x1, x2_warp)                                  # model.py:83
        if args.corr_activation: F.leaky_relu_(corr)                   # model.py:84
        ... torch.cat([x1, corr, flow], dim = 1) ...                   # model.py:89/91
    becomes
        inp = self.corr_cat(x1, x2_warp, flow)

    The correlation kernels write straight into the concatenated buffer's corr channels
    (with the leaky_relu fused when ``corr_activation``); ctor as ``Correlation``."""

    def __init__(self, pad_size=9, kernel_size=1, max_displacement=9, stride1=1, stride2=2,
                 corr_multiply=1, corr_activation=False, negative_slope=0.01):
        super().__init__()
        self.params = (pad_size, kernel_size, max_displacement, stride1, stride2)
        self.negative_slope = negative_slope if corr_activation else None

    def forward(self, x1, x2_warp, flow):
        return CorrelationCatFunction.apply(x1, x2_warp, flow, *self.params,
                                            self.negative_slope)


class UpsampleWarp(nn.Module):
    """model.py:78 + :80 in one call:

        flow = F.upsample(flow, scale_factor=2, mode='bilinear') * 2     # model.py:78
        x2_warp = self.warping_layer(x2, flow)                            # model.py:80
    becomes
        x2_warp, flow = self.upsample_warp(x2, flow)

    torch 0.4's bilinear upsample (align_corners=False) and the WarpingLayer chain
    (align_corners=True grid_sample); gradients flow to x2 and the coarse flow.
    """

    def forward(self, x2, flow_coarse):
        return UpsampleWarpFunction.apply(x2, flow_coarse)


class CostVolumeLayer(nn.Module):
    """modules.py:45-74: (2*search_range+1)^2 channels in the reference's order, / K."""

    def __init__(self, args):
        super().__init__()
        self.args = args
        self.search_range = args.search_range

    def forward(self, src, tgt):
        return _library.cost_volume(src, tgt, self.search_range)


# ---------------------------------------------------------------------------------------
# feature operators (features.py): functions and modules
# ---------------------------------------------------------------------------------------
_PLAIN = (torch.Tensor, nn.Parameter)
_functorch = torch._C._functorch
_level, _trace = _functorch.peek_interpreter_stack, torch._C._get_tracing_state
_modes = torch._C._len_torch_dispatch_stack


def _traced(*tensors):
    """Tracers, subclasses and torch.func see one opaque torch.ops.pwcnet node; eager calls go
    straight to the kernels.  (The question takes 0.4 us of the host.)"""
    if torch.compiler.is_compiling():
        return True
    if _level() is not None:
        # (a node without a forward-mode formula would give zeros)
        if any(i.key() == _functorch.TransformType.Jvp for i in _functorch.get_interpreter_stack()):
            raise RuntimeError("pwcnet_amd: the feature operators have no forward-mode derivatives")
        return True
    if _trace() is not None or _modes() > 0:  # torch.jit.trace; a dispatch mode
        return True
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            return True
    return False


def layer_norm(x, weight=None, bias=None, eps=1e-5, channel_dim=1):
    """(x - mean) / sqrt(var + eps) * weight + bias over the channels of each pixel of a map
    [B, C, *spatial] (``channel_dim=1``) or of each token [..., C] (``channel_dim=-1``)."""
    if _traced(x, weight, bias):
        return _library.layer_norm(x, weight, bias, eps, channel_dim)[0]
    return _features._ext.layer_norm(x, weight, bias, eps, channel_dim)


def rotary(x, inv_freq, axis, positions=None, grid=None, origin=None, interleaved=False):
    """x [B, N, heads, D] with its channel pairs turned by position[axis[j]] * inv_freq[j]; see
    ``features.rotary_forward``.  ``inv_freq`` and ``axis`` come from ``rotary_frequencies``."""
    if _traced(x, inv_freq, axis, positions):
        if _trace() is not None:  # its sizes are no ints: they stay as traced
            grid, origin = (v and [int(n) for n in v] for v in (grid, origin))
        grid = None if grid is None else list(grid)
        origin = None if origin is None else list(origin)
        return _library.rotary(x, inv_freq, axis, positions, grid, origin, interleaved, False)
    return _features._ext.rotary(x, inv_freq, axis, positions, grid, origin, interleaved)


def linear(x, weight, bias=None, residual=None, activation="none", negative_slope=0.1,
           channel_dim=1):
    """act(x W^T + bias) + residual over x's channels: on maps a 1x1 convolution with its
    activation and skip in one kernel.  ``activation``: one of ``features.ACTIVATIONS``.  How the
    16-bit backward pass rounds: ``features.linear_backward``."""
    activation = activation or "none"
    if _traced(x, weight, bias, residual):
        return _library.linear(x, weight, bias, residual, activation, negative_slope, channel_dim)
    return _features._ext.linear(x, weight, bias, residual, activation, negative_slope,
                                 channel_dim)


def gated_linear(x, weight, bias=None, activation="silu", negative_slope=0.1, channel_dim=1):
    """act(x Wg^T + bg) * (x Wu^T + bu) over x's channels, weight = [Wg; Wu]: both projections,
    the activation and the product in one kernel.  How the 16-bit backward pass rounds:
    ``features.linear_backward``."""
    activation = activation or "none"
    if _traced(x, weight, bias):
        return _library.gated_linear(x, weight, bias, activation, negative_slope, channel_dim)
    return _features._ext.gated_linear(x, weight, bias, activation, negative_slope, channel_dim)


class LayerNorm(nn.Module):
    """``layer_norm`` with a weight (ones) and, unless ``bias=False``, a bias (zeros)."""

    def __init__(self, channels, eps=1e-5, bias=True, channel_dim=1):
        super().__init__()
        self.eps, self.channel_dim = eps, channel_dim
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps, self.channel_dim)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}, channel_dim={self.channel_dim}"


class RotaryPosition(nn.Module):
    """Rotary positions for maps [B, heads * D, *spatial] (``channel_dim=1``) or tokens
    [B, N, heads, D] (``channel_dim=-1``).

    ``sections``: channel pairs of each axis, the last spatial axis last; axes before the map's
    own (a frame's time) are constants of the call's ``origin``.  Tokens need ``positions``."""

    def __init__(self, sections, heads=1, base=10000.0, shared=False, interleaved=False,
                 channel_dim=1):
        super().__init__()
        if channel_dim not in (1, -1):
            raise ValueError(f"RotaryPosition: channel_dim {channel_dim} is neither 1 nor -1")
        inv_freq, axis = _features.rotary_frequencies(sections, base, shared)
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self.register_buffer("axis", axis, persistent=False)
        self.sections, self.heads = tuple(sections), heads
        self.interleaved, self.channel_dim = interleaved, channel_dim

    def _apply(self, fn, recurse=True):
        # angles stay in 64 bits when the module is cast: only the device follows
        kept = self.inv_freq
        super()._apply(fn, recurse)
        if self.inv_freq.dtype != torch.float64:
            self.inv_freq = kept.to(self.inv_freq.device)
        return self

    def forward(self, x, positions=None, origin=None):
        if self.channel_dim == -1:
            if origin is not None:
                raise ValueError("RotaryPosition: tokens stand at their positions; origin belongs "
                                 "to maps")
            return rotary(x, self.inv_freq, self.axis, positions, interleaved=self.interleaved)
        spatial, axes = tuple(x.shape[2:]), len(self.sections)
        if x.dim() < 3 or len(spatial) > axes or x.shape[1] % self.heads:
            raise ValueError(f"RotaryPosition: map {tuple(x.shape)} for {axes} axes and "
                             f"{self.heads} heads")
        B, C = x.shape[:2]
        n = math.prod(spatial)
        v = x.reshape(B, self.heads, C // self.heads, n).permute(0, 3, 1, 2)
        grid = None if positions is not None else (1,) * (axes - len(spatial)) + spatial
        y = rotary(v, self.inv_freq, self.axis, positions, grid, origin, self.interleaved)
        return y.permute(0, 2, 3, 1).reshape(x.shape)

    def extra_repr(self):
        return f"{self.sections}, heads={self.heads}, channel_dim={self.channel_dim}"


class ChannelLinear(nn.Module):
    """``linear`` with its weight [out, in] and bias; on maps a 1x1 convolution."""

    def __init__(self, in_channels, out_channels, bias=True, activation="none",
                 negative_slope=0.1, channel_dim=1):
        super().__init__()
        self.activation, self.negative_slope = activation, negative_slope
        self.channel_dim = channel_dim
        self.weight = nn.Parameter(torch.empty(out_channels, in_channels))
        nn.init.xavier_uniform_(self.weight)
        self.bias = nn.Parameter(torch.zeros(out_channels)) if bias else None

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, residual, self.activation, self.negative_slope,
                      self.channel_dim)

    def extra_repr(self):
        return f"{self.weight.shape[1]}, {self.weight.shape[0]}, activation={self.activation!r}"


class GatedLinear(nn.Module):
    """``gated_linear`` with its weight [gate; up] of 2 * hidden rows and bias."""

    def __init__(self, in_channels, hidden_channels, bias=True, activation="silu",
                 negative_slope=0.1, channel_dim=1):
        super().__init__()
        self.activation, self.negative_slope = activation, negative_slope
        self.channel_dim = channel_dim
        self.weight = nn.Parameter(torch.empty(2 * hidden_channels, in_channels))
        for half in self.weight.chunk(2):
            nn.init.xavier_uniform_(half)
        self.bias = nn.Parameter(torch.zeros(2 * hidden_channels)) if bias else None

    def forward(self, x):
        return gated_linear(x, self.weight, self.bias, self.activation, self.negative_slope,
                            self.channel_dim)

    def extra_repr(self):
        return (f"{self.weight.shape[1]}, {self.weight.shape[0] // 2}, "
                f"activation={self.activation!r}")


class FeatureBlock(nn.Module):
    """x + project(gated(norm(x))) over the channels of a map: three kernels forward, the skip in
    the last one's epilogue."""

    def __init__(self, channels, hidden_channels=None, activation="silu", channel_dim=1):
        super().__init__()
        hidden = hidden_channels or 2 * channels
        self.norm = LayerNorm(channels, channel_dim=channel_dim)
        self.gated = GatedLinear(channels, hidden, activation=activation, channel_dim=channel_dim)
        self.project = ChannelLinear(hidden, channels, channel_dim=channel_dim)

    def forward(self, x):
        return self.project(self.gated(self.norm(x)), residual=x)


def get_grid(x: torch.Tensor) -> torch.Tensor:
    """utils.py:3-8: B x 2 x H x W grid of linspace(-1, 1) (x then y)."""
    B, _, H, W = x.shape
    horiz = torch.linspace(-1.0, 1.0, W).view(1, 1, 1, W).expand(B, 1, H, W)
    vert = torch.linspace(-1.0, 1.0, H).view(1, 1, H, 1).expand(B, 1, H, W)
    return torch.cat([horiz, vert], 1)
