"""Feature operators over the C ABI: layer norm, rotary positions, linear and gated linear -- what a
model puts between the feature pyramid and the correlation.

Each works on feature maps ``[B, C, *spatial]`` (``channel_dim=1``) and on tokens ``[..., C]``
(``channel_dim=-1``), fp32, fp16 or bf16 storage with fp32 sums, on the current stream of the
tensors' device.  Nothing synchronises; workspaces come from the caching allocator per call.

Argument checks, allocation and the autograd nodes are native (csrc/bind_features.cpp, module
``_features_ext``): the smallest calls are a few microseconds of GPU work.  ``layer_norm``,
``rotary``, ``linear`` and ``gated_linear`` of the package are differentiable; the functions here
with ``_forward`` and ``_backward`` in their names are the passes alone.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

try:
    from . import _features_ext as _ext
except ImportError as _why:  # not built, or built against another torch
    class _Missing:
        def __init__(self, why):
            self._why = why

        def __getattr__(self, name):
            raise _lib.HipLibraryMissing(
                f"pwcnet_amd: _features_ext is not built ({self._why}); run `make -C "
                "pwc-net_pytorch_amd/csrc` or `python -c 'import __graft_entry__ as g; "
                "g.build()'`")

    _ext = _Missing(_why)

MAP, TOKENS = 0, 1
ACTIVATIONS = {"none": 0, "relu": 1, "leaky_relu": 2, "sigmoid": 3, "tanh": 4, "silu": 5,
               "gelu": 6, "gelu_tanh": 7}


def _bind():
    """Give the module the C entries' addresses (it asks at its first call)."""
    lib = _lib.load()
    _ext.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
               for name in _ext.entries()})


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, channel_dim=1, stats=False):
    """(y, mean, rstd); mean and rstd (fp32, one a token) are None unless ``stats``."""
    return _ext.layer_norm_forward(x, weight, bias, eps, channel_dim, stats)


def layer_norm_backward(x, weight, grad_out, mean, rstd, channel_dim=1, needs=(True, True, True)):
    """(grad_x, grad_weight, grad_bias), None where ``needs`` says so."""
    return _ext.layer_norm_backward(x, weight, grad_out, mean, rstd, channel_dim, needs)


def rotary_frequencies(sections, base=10000.0, shared=False, device=None):
    """(inv_freq, axis) for ``sections`` pairs of each axis, in order: frequencies base^(-j / n)
    with j and n counted within the axis, or (``shared``) over all pairs."""
    sections = [int(s) for s in sections]
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) == 0:
        raise ValueError(f"rotary: sections {sections}: pairs for one to four axes")
    total = sum(sections)
    j = [torch.arange(s, dtype=torch.float64) / s for s in sections]
    at = torch.arange(total, dtype=torch.float64) / total if shared else torch.cat(j)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.int32)
    return (float(base) ** -at).to(device), axis.to(device)


def rotary_forward(x, inv_freq, axis, positions=None, grid=None, origin=None, interleaved=False,
                   inverse=False):
    """x [B, N, heads, D] (any strides) with pair j of each head's channels -- (j, R + j), or
    (2j, 2j + 1) where ``interleaved`` -- turned by position[axis[j]] * inv_freq[j].

    ``inv_freq``: fp64 [R]; ``axis``: int32 [R] of the positions' axes (values outside are taken to
    the nearest).  ``positions``: [N, A], [1, N, A] or [B, N, A] (int32, int64 or fp32), or None:
    tokens stand at their raster places in ``grid`` (A sizes) plus ``origin``.  Channels from 2 R
    on pass.  ``inverse`` turns back."""
    return _ext.rotary_forward(x, inv_freq, axis, positions, grid, origin, interleaved, inverse)


def linear_forward(x, weight, bias=None, residual=None, activation="none", negative_slope=0.1,
                   channel_dim=1):
    """act(x W^T + b) + residual over x's channels; weight [O, K]."""
    return _ext.linear_forward(x, weight, bias, residual, activation, negative_slope, channel_dim)


def linear_backward(x, weight, bias, grad_out, activation="none", negative_slope=0.1,
                    channel_dim=1, needs=(True, True, True)):
    """(grad_x, grad_weight, grad_bias), None where ``needs`` says so; the residual's gradient is
    grad_out itself.

    With an activation the gradient of the sums is kept in x's type between the products: in small
    16-bit calls (at most 0.5 GFLOP a product, 2 * tokens * out * in, by the kernels of small tiles)
    as a value and what its rounding took, in others as a value alone, which makes the gradients'
    error 1.4 times that of their own rounding.  In fp16 it is infinite beyond 65504 and nothing below 2^-25, as between the layers
    of an fp16 program: scale the loss."""
    return _ext.linear_backward(x, weight, bias, grad_out, activation, negative_slope, channel_dim,
                                needs)


def gated_linear_forward(x, weight, bias=None, activation="silu", negative_slope=0.1,
                         channel_dim=1):
    """act(x Wg^T + bg) * (x Wu^T + bu) over x's channels; weight [2 O, K] = [Wg; Wu]."""
    return _ext.gated_linear_forward(x, weight, bias, activation, negative_slope, channel_dim)


def gated_linear_backward(x, weight, bias, grad_out, activation="silu", negative_slope=0.1,
                          channel_dim=1, needs=(True, True, True)):
    """(grad_x, grad_weight, grad_bias), None where ``needs`` says so; the gradient of the sums is
    kept as in ``linear_backward`` (counting both projections' rows)."""
    return _ext.gated_linear_backward(x, weight, bias, grad_out, activation, negative_slope,
                                      channel_dim, needs)
