"""CPU: the feature operators' refusals, at the Python functions and at the C entries (no call here
reaches a device), their frequencies, modules and shapes under tracing."""
import ctypes

import pytest
import torch

LIM = 2 ** 31


def _lib():
    from pwcnet_amd import _lib
    return _lib.load()


def _refused(ret, text):
    assert ret == 0
    assert text.encode() in _lib().pwc_last_error(), _lib().pwc_last_error()


def test_layer_norm_entry_refuses():
    lib, p, z = _lib(), ctypes.c_void_p(64), None

    def fwd(x=p, y=p, mean=z, rstd=z, layout=0, B=1, P=4, C=8, stride=32, eps=1e-5, dtype=0):
        return lib.pwc_layer_norm_forward(x, z, z, y, mean, rstd, layout, B, P, C, stride, eps,
                                          dtype, z)

    _refused(fwd(dtype=7), "unsupported dtype")
    _refused(fwd(layout=2), "unknown layout")
    _refused(fwd(B=-1), "negative dimension")
    _refused(fwd(C=0), "no channels")
    _refused(fwd(layout=1, B=2), "tokens have one batch")
    _refused(fwd(P=LIM), "too large")
    _refused(fwd(B=2, stride=31), "stride smaller")
    _refused(fwd(layout=1, stride=7), "stride smaller")
    _refused(fwd(layout=1, stride=0), "stride smaller")
    _refused(fwd(eps=-1.0), "eps")
    _refused(fwd(eps=float("nan")), "eps")
    _refused(fwd(mean=p), "mean and rstd")
    _refused(fwd(x=z), "null")
    _refused(fwd(y=z), "null")
    assert fwd(x=z, y=z, B=0) == 1 and fwd(x=z, y=z, P=0) == 1

    def bwd(x=p, dy=p, mean=p, gx=p, gw=p, gb=p, ws=p, n=1 << 20, B=1, P=4, dtype=0):
        return lib.pwc_layer_norm_backward(x, z, dy, mean, p, gx, gw, gb, 0, B, P, 8, 32, dtype,
                                           ws, n, z)

    _refused(bwd(dtype=-1), "unsupported dtype")
    _refused(bwd(x=z), "null")
    _refused(bwd(dy=z), "null")
    _refused(bwd(mean=z), "null")
    _refused(bwd(n=8), "workspace too small")
    _refused(bwd(ws=z), "workspace too small")
    assert bwd(gx=z, gw=z, gb=z) == 1
    assert bwd(gw=z, gb=z, B=0) == 1
    assert lib.pwc_layer_norm_backward_workspace_size(0, 1, 4, 8, 0) >= 64
    assert lib.pwc_layer_norm_backward_workspace_size(0, 1, -4, 8, 0) == 0


def test_product_entries_refuse():
    lib, p, z = _lib(), ctypes.c_void_p(64), None

    def fwd(x=p, w=p, y=p, layout=0, B=1, P=4, K=8, O=6, stride=32, act=0, dtype=0, gated=False):
        geo = (layout, B, P, K, O, stride, act, 0.1, dtype, z, 0, z)
        return (lib.pwc_gated_linear_forward(x, w, z, y, *geo) if gated
                else lib.pwc_linear_forward(x, w, z, z, y, *geo))

    for gated in (False, True):
        _refused(fwd(dtype=3, gated=gated), "unsupported dtype")
        _refused(fwd(layout=-1, gated=gated), "unknown layout")
        _refused(fwd(P=-4, gated=gated), "negative dimension")
        _refused(fwd(K=0, gated=gated), "no channels")
        _refused(fwd(O=0, gated=gated), "output channels")
        _refused(fwd(O=LIM - 1, gated=gated), "output channels")
        _refused(fwd(act=8, gated=gated), "unknown activation")
        _refused(fwd(act=-1, gated=gated), "unknown activation")
        _refused(fwd(layout=1, B=3, gated=gated), "tokens have one batch")
        _refused(fwd(B=2, stride=31, gated=gated), "stride smaller")
        _refused(fwd(B=LIM - 1, P=2, K=1, stride=2, gated=gated), "too large")
        _refused(fwd(x=z, gated=gated), "null")
        _refused(fwd(w=z, gated=gated), "null")
        _refused(fwd(y=z, gated=gated), "null")
        assert fwd(x=z, w=z, y=z, P=0, gated=gated) == 1

        def bwd(x=p, w=p, dy=p, gx=p, gw=p, gb=p, ws=p, n=1 << 24, P=4, act=5, dtype=0):
            geo = (0, 1, P, 8, 6, 32, act, 0.1, dtype, ws, n, z)
            return (lib.pwc_gated_linear_backward if gated else lib.pwc_linear_backward)(
                x, w, z, dy, gx, gw, gb, *geo)

        _refused(bwd(dtype=9), "unsupported dtype")
        _refused(bwd(act=99), "unknown activation")
        _refused(bwd(x=z), "null")
        _refused(bwd(w=z), "null")
        _refused(bwd(dy=z), "null")
        _refused(bwd(n=16), "workspace too small")
        _refused(bwd(ws=z), "workspace too small")
        assert bwd(gx=z, gw=z, gb=z) == 1
        assert bwd(gw=z, gb=z, P=0) == 1
    back, gated = lib.pwc_linear_backward_workspace_size, lib.pwc_gated_linear_backward_workspace_size
    assert back(p, p, p, 0, 1, 4, 8, 6, 32, 0, 9) == 0
    assert gated(p, p, p, 0, 1, 4, 0, 6, 32, 0) == 0
    # dz [4, 12], and the sums of dW [12, 8] where k is split
    assert gated(p, p, p, 0, 1, 4, 8, 6, 32, 0) >= 4 * 12 * 4
    assert gated(p, p, p, 0, 1, 10 ** 6, 8, 6, 8 * 10 ** 6, 0) >= 10 ** 6 * 12 * 4 + 2 * 12 * 8 * 4
    # large 16-bit products are given rows at 16-byte places: x, W (and dz) where theirs are not
    fwd = lib.pwc_linear_forward_workspace_size
    odd = ctypes.c_void_p(66)
    assert fwd(p, p, 1, 1, 4096, 1024, 1024, 1024, 2) == 0
    assert fwd(odd, p, 1, 1, 4096, 1024, 1024, 1024, 2) == 4096 * 1024 * 2
    assert fwd(p, odd, 1, 1, 4096, 1024, 1024, 1024, 2) == 1024 * 1024 * 2
    assert fwd(p, p, 1, 1, 4096, 1024, 1024, 1025, 2) == 4096 * 1024 * 2
    assert fwd(p, p, 1, 1, 4096, 1023, 1024, 1023, 2) == (4096 + 1024) * 1024 * 2
    assert fwd(p, p, 1, 1, 4096, 1023, 1024, 1023, 0) == (4096 + 1024) * 1024 * 4
    assert fwd(p, p, 1, 1, 100, 99, 98, 99, 2) == 0
    assert fwd(p, p, 1, 1, 16, 9999, 9999, 9999, 2) == 0  # a pass over W reads it as it lies
    _refused(lib.pwc_linear_forward(p, p, z, z, p, 1, 1, 4096, 1023, 1024, 1023, 0, 0.1, 2, z, 0,
                                    z), "workspace too small")
    _refused(lib.pwc_linear_forward(p, p, z, z, p, 1, 1, 4096, 1023, 1024, 1023, 0, 0.1, 2, p,
                                    1 << 30, z), "workspace not aligned")


def test_rotary_entry_refuses():
    from pwcnet_amd import _lib as L
    lib, p, z = _lib(), ctypes.c_void_p(64), None

    def call(x=p, y=p, at=z, dtype=0, shape=True, **kw):
        s = L.RotaryShape(B=1, N=6, heads=2, D=8, pairs=4, axes=2)
        s.grid = (ctypes.c_longlong * 4)(2, 3)
        for k, v in kw.items():
            setattr(s, k, (ctypes.c_longlong * 4)(*v) if isinstance(v, tuple) else v)
        return lib.pwc_rotary(x, y, at, p, p, ctypes.byref(s) if shape else None, 0, dtype, z)

    _refused(call(dtype=5), "unsupported dtype")
    _refused(call(shape=False), "null shape")
    _refused(call(B=-1), "negative dimension")
    _refused(call(N=LIM), "too large")
    _refused(call(heads=1 << 21), "too large")
    _refused(call(pairs=5), "more pairs")
    _refused(call(pairs=-1), "more pairs")
    _refused(call(axes=0), "axes")
    _refused(call(axes=5), "axes")
    _refused(call(grid=(2, 2)), "grid")
    _refused(call(grid=(LIM, LIM)), "grid")
    _refused(call(grid=(-2, -3)), "grid")
    _refused(call(origin=(2 ** 60, 0)), "origin")
    _refused(call(at=p, position_type=3), "position type")
    _refused(call(x=z), "null")
    _refused(call(y=z), "null")
    assert call(x=z, y=z, B=0) == 1
    assert call(x=z, y=z, N=0, grid=(0, 3)) == 1


def test_functions_refuse_host_tensors_and_bad_arguments():
    import pwcnet_amd as P
    x = torch.zeros(2, 4, 3, 3)
    w = torch.zeros(6, 4)
    f, a = P.rotary_frequencies((2,))
    for call in (lambda: P.layer_norm(x), lambda: P.linear(x, w), lambda: P.gated_linear(x, w),
                 lambda: P.rotary(x, f, a, grid=(4,)), lambda: P.LayerNorm(4)(x),
                 lambda: P.FeatureBlock(4)(x), lambda: P.RotaryPosition((1, 1))(x)):
        with pytest.raises(RuntimeError, match="HIP"):
            call()
    with pytest.raises(ValueError, match="no gradient"):
        P.rotary(x, f, a, torch.zeros(4, 1, requires_grad=True))
    for bad in ((), (1, 2, 3, 4, 5), (0,), (-1, 3)):
        with pytest.raises(ValueError):
            P.rotary_frequencies(bad)
    with pytest.raises(ValueError, match="channel_dim"):
        P.RotaryPosition((2,), channel_dim=2)
    with pytest.raises(ValueError, match="axes"):
        P.RotaryPosition((2,))(x)


def test_geometry():
    """How shapes and strides are taken, on host tensors: (taken as is, layout, B, P, C, stride)."""
    from pwcnet_amd import features as F
    by_rows, matrix = F._ext.by_rows, F._ext.matrix
    for dim in (0, 2, -2):
        with pytest.raises(ValueError, match="channel_dim"):
            by_rows((2, 3, 4, 5), dim, "x")
    assert by_rows((2, 3, 4, 5), 3, "x")
    for shape in ((3,), ()):
        with pytest.raises(ValueError, match="channel_dim"):
            by_rows(shape, 1, "x")
    assert by_rows((3,), -1, "x") and by_rows((5, 3), 1, "x")
    assert not by_rows((5, 3, 2), 1, "x")
    base = torch.zeros(6, 10, 12)
    for t, stride in ((base, 12), (base[..., :8], 12), (base[:, 2:3], 120), (base[:1, ::2], 24),
                      (base.transpose(0, 1), None), (base[..., ::2], None),
                      (base[:, :5, :7], None), (torch.zeros(1, 12).expand(4, 12), None),
                      (torch.zeros(4, 1).expand(4, 1), 1), (torch.zeros(4, 2)[:, :1], 2)):
        got = matrix(t, True)
        assert got == (stride is not None, F.TOKENS, 1, t.numel() // t.shape[-1], t.shape[-1],
                       t.shape[-1] if stride is None else stride)
    for t, stride in ((base, 120), (base[:, 2:7], 120), (base[::2], 240),
                      (base.transpose(1, 2), None), (base[..., 1:], None),
                      (base[:1].expand(3, 10, 12), None)):
        got = matrix(t, False)
        assert got == (stride is not None, F.MAP, t.shape[0], t.shape[2], t.shape[1],
                       t.shape[1] * t.shape[2] if stride is None else stride)


def test_frequencies():
    import pwcnet_amd as P
    f, a = P.rotary_frequencies((2, 4), base=100.0)
    assert a.tolist() == [0, 0, 1, 1, 1, 1] and f.dtype == torch.float64
    want = torch.tensor([1, 100 ** -0.5, 1, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75],
                        dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-15, atol=0)
    f, _ = P.rotary_frequencies((2, 4), base=100.0, shared=True)
    assert torch.allclose(f, 100.0 ** -(torch.arange(6, dtype=torch.float64) / 6), rtol=1e-14,
                          atol=0)
    m = P.RotaryPosition((2, 4)).to(torch.bfloat16)
    assert m.inv_freq.dtype == torch.float64 and not m.state_dict()


def test_traced_as_single_nodes():
    """Under tracing each operator is one torch.ops.pwcnet node with the right shape."""
    import pwcnet_amd as P
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(2, 8, 5, 6)
        w = torch.empty(12, 8)
        assert P.layer_norm(x).shape == x.shape
        assert P.linear(x, w).shape == (2, 12, 5, 6)
        assert P.gated_linear(x, w).shape == (2, 6, 5, 6)
        assert P.linear(x.reshape(-1, 8), w, channel_dim=-1).shape == (60, 12)
        assert P.RotaryPosition((2, 2))(x).shape == x.shape
        assert P.FeatureBlock(8)(x).shape == x.shape


def test_net_is_unchanged_without_refined_features():
    from pwcnet_amd.net import Net, NetArgs
    torch.manual_seed(5)
    a = Net(NetArgs())
    torch.manual_seed(5)
    b = Net(NetArgs(feature_blocks=1, feature_rotary=True))
    extra = set(b.state_dict()) - set(a.state_dict())
    assert len(extra) == 5 * 6 and all(k.startswith("FeatureBlocks(Lv") for k in extra)
    assert all(torch.equal(v, b.state_dict()[k]) for k, v in a.state_dict().items())
    assert a.refine([1, 2], 0) == [1, 2]
    assert [m.sections for m in b.feature_rotaries] == [
        (24, 36, 36), (16, 24, 24), (12, 18, 18), (8, 12, 12), (4, 6, 6)]
