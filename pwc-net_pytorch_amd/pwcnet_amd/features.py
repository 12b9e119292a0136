"""Feature operators over the C ABI plus their autograd Functions: layer norm, rotary positions,
linear and gated linear -- what a model puts between the feature pyramid and the correlation.

Each works on feature maps ``[B, C, *spatial]`` (``channel_dim=1``) and on tokens ``[..., C]``
(``channel_dim=-1``), fp32, fp16 or bf16 storage with fp32 sums, on the current stream of the
tensors' device.  Nothing synchronises; workspaces come from the caching allocator per call.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _i32, _nullctx, _ptr, _stream, _workspace

MAP, TOKENS = 0, 1
ACTIVATIONS = {"none": 0, "relu": 1, "leaky_relu": 2, "sigmoid": 3, "tanh": 4, "silu": 5,
               "gelu": 6, "gelu_tanh": 7}
_POSITION_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}
_NULL = ctypes.c_void_p(0)


def _check(what, *ts):
    """Device, dtype and kind of the tensors that are there (None is skipped)."""
    first = ts[0]
    for t in ts:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {type(t)}")
        if t.device.type != "cuda":
            raise RuntimeError(f"{what}: pwcnet_amd runs on HIP devices only (got a {t.device} "
                               "tensor); there is no CPU implementation")
        if t.device != first.device:
            raise RuntimeError(f"{what}: tensors on different devices ({t.device} vs "
                               f"{first.device})")
        if t.dtype not in _lib.DTYPE_CODES:
            raise TypeError(f"{what}: unsupported dtype {t.dtype}")
        if t.dtype != first.dtype:
            raise TypeError(f"{what}: mixed dtypes {t.dtype} vs {first.dtype}")


def _opt(t):
    return _NULL if t is None else _ptr(t)


def _on(t):
    return torch.cuda.device(t.device) if t.is_cuda else _nullctx()


def _by_rows(shape, channel_dim, what):
    """True if ``shape`` is taken as tokens [..., C], False as a map [B, C, *spatial]."""
    n = len(shape)
    if n < 1 or channel_dim not in (1, -1, n - 1) or (channel_dim == 1 and n < 2):
        raise ValueError(f"{what}: channel_dim {channel_dim} of a tensor of shape {tuple(shape)} "
                         "(1 for maps [B, C, *spatial], -1 for tokens [..., C])")
    return channel_dim != 1 or n == 2


def _matrix(x, rows):
    """(x, layout, B, P, C, stride): x as the C ABI takes it, copied only where its strides are
    not those of tokens / images a fixed distance apart."""
    if rows:
        C = x.shape[-1]
        P = x.numel() // C if C else 0
        stride = C
        if not x.is_contiguous():
            stride = _row_stride(x, C)
            if stride is None:
                x, stride = x.contiguous(), C
        return x, TOKENS, 1, P, C, stride
    B, C = x.shape[:2]
    P = 1
    for s in x.shape[2:]:
        P *= s
    stride = C * P
    if not x.is_contiguous():
        if x.numel() and x.stride(0) >= C * P and x[0].is_contiguous():
            stride = x.stride(0)
        else:
            x = x.contiguous()
    return x, MAP, B, P, C, stride


def _row_stride(x, C):
    """The distance of x's tokens if its leading dimensions are one, else None."""
    if x.numel() == 0 or (C > 1 and x.stride(-1) != 1):
        return None
    stride, span = None, 0
    for size, st in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride, span = st, st * size
        elif st != span:
            return None
        else:
            span = st * size
    if stride is None:
        return C
    return stride if stride >= C else None


def _vector(what, name, v, n):
    if v is None:
        return None
    if tuple(v.shape) != (n,):
        raise ValueError(f"{what}: {name} shape {tuple(v.shape)} != {(n,)}")
    return v.contiguous()


# ---------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------
def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, channel_dim=1, stats=False):
    """(y, mean, rstd); mean and rstd (fp32, one a token) are None unless ``stats``."""
    _check("LayerNorm", x, weight, bias)
    rows = _by_rows(x.shape, channel_dim, "LayerNorm")
    shape = x.shape
    x, layout, B, P, C, stride = _matrix(x, rows)
    if C == 0:
        raise ValueError("LayerNorm: no channels")
    if not eps >= 0:
        raise ValueError(f"LayerNorm: eps {eps} is negative")
    weight = _vector("LayerNorm", "weight", weight, C)
    bias = _vector("LayerNorm", "bias", bias, C)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean = torch.empty(B * P, dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    if y.numel():
        _lib.check(_lib.load().pwc_layer_norm_forward(
            _ptr(x), _opt(weight), _opt(bias), _ptr(y), _opt(mean), _opt(rstd), layout, B, P, C,
            stride, eps, _lib.DTYPE_CODES[x.dtype], _stream(x.device)), "LayerNorm_forward")
    return y, mean, rstd


def layer_norm_backward(x, weight, grad_out, mean, rstd, channel_dim=1, needs=(True, True, True)):
    """(grad_x, grad_weight, grad_bias), None where ``needs`` says so."""
    _check("LayerNorm backward", x, weight, grad_out)
    if grad_out.shape != x.shape:
        raise ValueError(f"LayerNorm backward: grad_output shape {tuple(grad_out.shape)} != "
                         f"{tuple(x.shape)}")
    shape = x.shape
    x, layout, B, P, C, stride = _matrix(x, _by_rows(shape, channel_dim, "LayerNorm backward"))
    for t in (mean, rstd):
        if t.shape != (B * P,) or t.dtype != torch.float32 or t.device != x.device:
            raise ValueError("LayerNorm backward: mean / rstd are not the forward pass's")
    grad_out = grad_out.contiguous()
    weight = _vector("LayerNorm backward", "weight", weight, C)
    gx = torch.empty(shape, dtype=x.dtype, device=x.device) if needs[0] else None
    gw, gb = (torch.empty(C, dtype=x.dtype, device=x.device) if n else None for n in needs[1:])
    lib, code = _lib.load(), _lib.DTYPE_CODES[x.dtype]
    nbytes = lib.pwc_layer_norm_backward_workspace_size(layout, B, P, C, code) \
        if gw is not None or gb is not None else 0
    ws, wsp = _workspace(nbytes, x.device)
    _lib.check(lib.pwc_layer_norm_backward(
        _ptr(x), _opt(weight), _ptr(grad_out), _ptr(mean), _ptr(rstd), _opt(gx), _opt(gw),
        _opt(gb), layout, B, P, C, stride, code, wsp, nbytes, _stream(x.device)),
        "LayerNorm_backward")
    del ws
    return gx, gw, gb


class LayerNormFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, channel_dim):
        with _on(x):
            y, mean, rstd = layer_norm_forward(x, weight, bias, eps, channel_dim, stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.channel_dim = channel_dim
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, mean, rstd = ctx.saved_tensors
        with _on(x):
            grads = layer_norm_backward(x, weight, grad, mean, rstd, ctx.channel_dim,
                                        ctx.needs_input_grad[:3])
        return (*grads, None, None)


# ---------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------
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

    ``positions``: [N, A], [1, N, A] or [B, N, A] (int32, int64 or fp32), or None: tokens stand at
    their raster places in ``grid`` (A sizes) plus ``origin``.  Channels from 2 R on pass.
    ``inverse`` turns back."""
    what = "rotary"
    _check(what, x)
    if x.dim() != 4:
        raise ValueError(f"{what}: expected [B, N, heads, D], got shape {tuple(x.shape)}")
    B, N, H, D = x.shape
    _i32(B, N, H, D)
    if inv_freq.dtype != torch.float64 or axis.dtype != torch.int32:
        raise TypeError(f"{what}: inv_freq is fp64 and axis int32, got {inv_freq.dtype} and "
                        f"{axis.dtype}")
    R = inv_freq.numel()
    if inv_freq.dim() != 1 or axis.shape != inv_freq.shape or 2 * R > D:
        raise ValueError(f"{what}: inv_freq {tuple(inv_freq.shape)} and axis "
                         f"{tuple(axis.shape)}: one value for each of at most {D // 2} pairs")
    s = _lib.RotaryShape(B=B, N=N, heads=H, D=D, pairs=R, interleaved=int(interleaved))
    if (positions is None) == (grid is None):
        raise ValueError(f"{what}: either positions or grid")
    if positions is not None:
        if origin is not None:
            raise ValueError(f"{what}: origin belongs to grid")
        if positions.dtype not in _POSITION_TYPES:
            raise TypeError(f"{what}: positions are int32, int64 or fp32, got {positions.dtype}")
        if positions.dim() not in (2, 3) or positions.shape[-2] != N or \
                (positions.dim() == 3 and positions.shape[0] not in (1, B)) or \
                not 1 <= positions.shape[-1] <= 4:
            raise ValueError(f"{what}: positions shape {tuple(positions.shape)} for {B} x {N} "
                             "tokens and one to four axes")
        s.axes, s.position_type = positions.shape[-1], _POSITION_TYPES[positions.dtype]
        shared = positions.dim() == 2 or positions.shape[0] == 1
        s.position_stride = (ctypes.c_longlong * 3)(
            0 if shared else positions.stride(0), positions.stride(-2), positions.stride(-1))
    else:
        grid = [int(g) for g in grid]
        origin = [0] * len(grid) if origin is None else [int(o) for o in origin]
        n = 1
        for g in grid:
            n *= g
        if not 1 <= len(grid) <= 4 or len(origin) != len(grid) or min(grid) < 0 or n != N:
            raise ValueError(f"{what}: grid {grid} and origin {origin} for {N} tokens")
        s.axes = len(grid)
        s.grid = (ctypes.c_longlong * 4)(*grid)
        s.origin = (ctypes.c_longlong * 4)(*origin)
    for t in (inv_freq, axis, positions):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{what}: tensors on different devices ({t.device} vs {x.device})")
    inv_freq, axis = inv_freq.contiguous(), axis.contiguous()
    y = torch.empty_like(x)
    s.x_stride = (ctypes.c_longlong * 4)(*x.stride())
    s.y_stride = (ctypes.c_longlong * 4)(*y.stride())
    if y.numel():
        _lib.check(_lib.load().pwc_rotary(
            _ptr(x), _ptr(y), _opt(positions), _ptr(inv_freq), _ptr(axis), ctypes.byref(s),
            int(inverse), _lib.DTYPE_CODES[x.dtype], _stream(x.device)), "rotary")
    return y


class RotaryFunction(Function):
    @staticmethod
    def forward(ctx, x, inv_freq, axis, positions, grid, origin, interleaved):
        ctx.save_for_backward(inv_freq, axis, positions)
        ctx.args = (grid, origin, interleaved)
        with _on(x):
            return rotary_forward(x, inv_freq, axis, positions, grid, origin, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        inv_freq, axis, positions = ctx.saved_tensors
        with _on(grad):
            g = rotary_forward(grad, inv_freq, axis, positions, *ctx.args, inverse=True)
        return (g,) + (None,) * 6


# ---------------------------------------------------------------------------------------
# linear and gated linear
# ---------------------------------------------------------------------------------------
def _activation(what, name):
    if name is None:
        name = "none"
    if name not in ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {name!r} (one of {sorted(ACTIVATIONS)})")
    return ACTIVATIONS[name]


def _product_args(what, x, weight, bias, channel_dim, gated):
    """The checked call: x, weight, bias as the C ABI takes them, its geometry and the output's
    shape."""
    rows = _by_rows(x.shape, channel_dim, what)
    ch = -1 if rows else 1
    if weight.dim() != 2 or weight.shape[1] != x.shape[ch] or weight.numel() == 0:
        raise ValueError(f"{what}: weight shape {tuple(weight.shape)} for {x.shape[ch]} channels")
    if gated and weight.shape[0] % 2:
        raise ValueError(f"{what}: weight [gate; up] has an odd number of rows "
                         f"({weight.shape[0]})")
    out = weight.shape[0] // 2 if gated else weight.shape[0]
    shape = list(x.shape)
    shape[ch] = out
    bias = _vector(what, "bias", bias, weight.shape[0])
    x, layout, B, P, K, stride = _matrix(x, rows)
    _i32(B * P, K, weight.shape[0])
    return x, weight.contiguous(), bias, (layout, B, P, K, out), stride, shape


def _product_backward(what, gated, x, weight, bias, grad_out, activation, negative_slope,
                      channel_dim, needs):
    _check(what, x, weight, bias, grad_out)
    code = _activation(what, activation)
    like = x.shape
    x, weight, bias, geo, stride, shape = _product_args(what, x, weight, bias, channel_dim, gated)
    if list(grad_out.shape) != shape:
        raise ValueError(f"{what}: grad_output shape {tuple(grad_out.shape)} != {tuple(shape)}")
    grad_out = grad_out.contiguous()
    gx = torch.empty(like, dtype=x.dtype, device=x.device) if needs[0] else None
    gw = torch.empty_like(weight) if needs[1] else None
    gb = torch.empty(weight.shape[0], dtype=x.dtype, device=x.device) if needs[2] else None
    lib, dt = _lib.load(), _lib.DTYPE_CODES[x.dtype]
    if gated:
        size = lib.pwc_gated_linear_backward_workspace_size(*geo, dt)
        call = lib.pwc_gated_linear_backward
    else:
        size = lib.pwc_linear_backward_workspace_size(*geo, code, dt)
        call = lib.pwc_linear_backward
    ws, wsp = _workspace(size, x.device)
    _lib.check(call(_ptr(x), _ptr(weight), _opt(bias), _ptr(grad_out), _opt(gx), _opt(gw),
                    _opt(gb), *geo, stride, code, float(negative_slope), dt, wsp, size,
                    _stream(x.device)), what)
    del ws
    return gx, gw, gb


def linear_forward(x, weight, bias=None, residual=None, activation="none", negative_slope=0.1,
                   channel_dim=1):
    """act(x W^T + b) + residual over x's channels; weight [O, K]."""
    what = "linear"
    _check(what, x, weight, bias, residual)
    code = _activation(what, activation)
    x, weight, bias, geo, stride, shape = _product_args(what, x, weight, bias, channel_dim, False)
    if residual is not None:
        if list(residual.shape) != shape:
            raise ValueError(f"{what}: residual shape {tuple(residual.shape)} != {tuple(shape)}")
        residual = residual.contiguous()
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    if y.numel():
        _lib.check(_lib.load().pwc_linear_forward(
            _ptr(x), _ptr(weight), _opt(bias), _opt(residual), _ptr(y), *geo, stride, code,
            float(negative_slope), _lib.DTYPE_CODES[x.dtype], _stream(x.device)), what)
    return y


def linear_backward(x, weight, bias, grad_out, activation="none", negative_slope=0.1,
                    channel_dim=1, needs=(True, True, True)):
    """(grad_x, grad_weight, grad_bias), None where ``needs`` says so; the residual's gradient is
    grad_out itself."""
    return _product_backward("linear backward", False, x, weight, bias, grad_out, activation,
                             negative_slope, channel_dim, needs)


def gated_linear_forward(x, weight, bias=None, activation="silu", negative_slope=0.1,
                         channel_dim=1):
    """act(x Wg^T + bg) * (x Wu^T + bu) over x's channels; weight [2 O, K] = [Wg; Wu]."""
    what = "gated_linear"
    _check(what, x, weight, bias)
    code = _activation(what, activation)
    x, weight, bias, geo, stride, shape = _product_args(what, x, weight, bias, channel_dim, True)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    if y.numel():
        _lib.check(_lib.load().pwc_gated_linear_forward(
            _ptr(x), _ptr(weight), _opt(bias), _ptr(y), *geo, stride, code, float(negative_slope),
            _lib.DTYPE_CODES[x.dtype], _stream(x.device)), what)
    return y


def gated_linear_backward(x, weight, bias, grad_out, activation="silu", negative_slope=0.1,
                          channel_dim=1, needs=(True, True, True)):
    """(grad_x, grad_weight, grad_bias), None where ``needs`` says so."""
    return _product_backward("gated_linear backward", True, x, weight, bias, grad_out, activation,
                             negative_slope, channel_dim, needs)


class LinearFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, negative_slope, channel_dim):
        ctx.save_for_backward(x, weight, bias)
        ctx.args = (activation, negative_slope, channel_dim)
        with _on(x):
            return linear_forward(x, weight, bias, residual, *ctx.args)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = (None, None, None)
        if any(need[:3]):
            with _on(x):
                grads = linear_backward(x, weight, bias, grad, *ctx.args, needs=need[:3])
        return (*grads, grad if need[3] else None, None, None, None)


class GatedLinearFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, negative_slope, channel_dim):
        ctx.save_for_backward(x, weight, bias)
        ctx.args = (activation, negative_slope, channel_dim)
        with _on(x):
            return gated_linear_forward(x, weight, bias, *ctx.args)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias = ctx.saved_tensors
        with _on(x):
            grads = gated_linear_backward(x, weight, bias, grad, *ctx.args,
                                          needs=ctx.needs_input_grad[:3])
        return (*grads, None, None, None)
