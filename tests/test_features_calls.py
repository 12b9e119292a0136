"""CPU: ways of calling the feature operators other than eagerly on plain tensors (no call here
reaches a device), and what the entries ask for."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import PKG


# ------------------------------------------------------------------------------- torch.jit.trace
def _operators():
    """(node name, a function of a map [B, 8, H, W] on any device)"""
    import pwcnet_amd as P
    w, b = torch.ones(12, 8), torch.zeros(12)
    return [("layer_norm", lambda x: P.layer_norm(x)),
            ("linear", lambda x: P.linear(x, w.to(x.device), b.to(x.device), activation="gelu")),
            ("gated_linear", lambda x: P.gated_linear(x, w.to(x.device))),
            ("rotary", P.RotaryPosition((2, 2)))]


@pytest.mark.filterwarnings("ignore")
def test_jit_trace_holds_the_nodes():
    """torch.jit.trace records each operator as its node, not the allocation of its output alone."""
    for name, call in _operators():
        traced = torch.jit.trace(call, torch.empty(2, 8, 5, 6, device="meta"), check_trace=False)
        kinds = [n.kind() for n in traced.graph.nodes()]
        assert f"pwcnet::{name}" in kinds, kinds
        assert not any(k in ("aten::empty", "aten::empty_like") for k in kinds), kinds
        x = torch.empty(3, 8, 5, 6, device="meta", requires_grad=True)
        y = traced(x)
        assert y.shape == (3, 6 if name == "gated_linear" else 12 if name == "linear" else 8, 5, 6)
        y.sum().backward()
        assert x.grad.shape == x.shape


def test_passes_refuse_jit_trace():
    """What torch.jit.trace cannot see is refused under it."""
    from pwcnet_amd import features as F
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    f, a = torch.ones(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32)
    for call in (lambda v: F.layer_norm_forward(v, channel_dim=-1)[0],
                 lambda v: F.linear_forward(v, w, channel_dim=-1),
                 lambda v: F.gated_linear_forward(v, w, channel_dim=-1),
                 lambda v: F.rotary_forward(v.view(1, 4, 1, 8), f, a, grid=(4,)),
                 lambda v: F.linear_backward(v, w, None, v, channel_dim=-1)[0]):
        with pytest.raises(RuntimeError, match="jit.trace"):
            torch.jit.trace(call, x, check_trace=False)


# ------------------------------------------------------------------------------- torch.func
def _calls(x, w, f, a):
    """The operators' functions of pwcnet_amd and the passes behind them, on tokens [N, 8]."""
    import pwcnet_amd as P
    from pwcnet_amd import features as F
    return ([lambda x, w: P.layer_norm(x, channel_dim=-1), lambda x, w: P.linear(x, w, channel_dim=-1),
             lambda x, w: P.gated_linear(x, w, channel_dim=-1),
             lambda x, w: P.rotary(x.view(1, -1, 1, 8), f, a, grid=(x.shape[0],))],
            [lambda x, w: F.layer_norm_forward(x, channel_dim=-1)[0],
             lambda x, w: F.linear_forward(x, w, channel_dim=-1),
             lambda x, w: F.gated_linear_forward(x, w, channel_dim=-1),
             lambda x, w: F.rotary_forward(x.view(1, -1, 1, 8), f, a, grid=(x.shape[0],))])


@pytest.mark.filterwarnings("ignore")
def test_wrapped_tensors_go_to_the_nodes():
    """vmap over any argument and a subclass in any place reach torch.ops.pwcnet; the passes alone
    refuse both."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w = torch.empty(3, 5, 8, device="meta"), torch.empty(3, 6, 8, device="meta")
    f, a = (torch.ones(4, dtype=torch.float64, device="meta"),
            torch.zeros(4, dtype=torch.int32, device="meta"))
    functions, passes = _calls(x, w, f, a)
    shapes = [(3, 5, 8), (3, 5, 6), (3, 5, 3), (3, 1, 5, 1, 8)]
    for call, shape in zip(functions, shapes):
        assert torch.vmap(call)(x, w).shape == shape
        assert torch.vmap(call, in_dims=(0, None))(x, w[0]).shape == shape
    for call, shape in zip(functions[1:3], shapes[1:3]):
        assert torch.vmap(call, in_dims=(None, 0))(x[0], w).shape == shape
    for call in passes:
        with pytest.raises(TypeError, match="plain tensors"):
            torch.vmap(call)(x, w)
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    fake = mode.from_tensor(torch.empty(6, 8))
    for call in functions[1:3]:
        assert type(call(torch.empty(5, 8), fake)) is type(fake)
    for call in passes[1:3]:
        with pytest.raises(TypeError, match="plain tensors"):
            call(fake, fake)


def test_forward_mode_is_refused_under_torch_func():
    """A node without a forward-mode formula would give zeros."""
    x, w = torch.empty(5, 8, device="meta"), torch.empty(6, 8, device="meta")
    f, a = (torch.ones(4, dtype=torch.float64, device="meta"),
            torch.zeros(4, dtype=torch.int32, device="meta"))
    for call in _calls(x, w, f, a)[0]:
        for run in (lambda: torch.func.jvp(lambda v: call(v, w), (x,), (x,)),
                    lambda: torch.func.jvp(lambda v: torch.vmap(lambda r: call(r[None], w))(v),
                                           (x,), (x,))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                run()


# ------------------------------------------------------------------------------- steps of k
_WALK = r"""
#include <cstdio>
#include <cstdlib>
#include "feat_steps.cuh"
// all blocks of one product: together they take every step once, and none past their ends
static long long walk(int segments, int K, int KS, int splits) {
  long long seen = 0;
  int seg = 0, k0 = 0;
  for (int z = 0; z < splits; ++z) {
    pwc::feat::Steps s;
    s.init(segments, K, KS, z, splits);
    const int mine = s.left;
    for (int n = 0; n < mine; ++n, s.next(K, KS)) {
      if (s.seg != seg || s.k0 != k0 || s.have(K) != K - k0 || s.have(K) <= 0) return -1;
      seen += s.have(K) < KS ? s.have(K) : KS;
      if (K - k0 > KS) k0 += KS; else k0 = 0, ++seg;
    }
    for (int n = 0; n < 5; ++n, s.next(K, KS))
      if (s.have(K) != 0) return -2;
  }
  return seg == segments && k0 == 0 ? seen : -3;
}
int main(int, char** v) { printf("%lld\n", walk(atoi(v[1]), atoi(v[2]), atoi(v[3]), atoi(v[4]))); }
"""


def test_steps_of_long_sums(tmp_path):
    """The product's walk over k, compiled for the host: every value once, nothing past the end, and
    no signed overflow (-ftrapv), up to the largest k that the entries take."""
    (tmp_path / "walk.cpp").write_text(_WALK)
    exe = str(tmp_path / "walk")
    subprocess.run(["g++", "-O1", "-ftrapv", "-I", os.path.join(PKG, "csrc"), "-o", exe,
                    str(tmp_path / "walk.cpp")], check=True)
    most = 2 ** 31 - 2 ** 16
    for segments, K, KS, splits in ((1, 1, 64, 1), (1, 64, 64, 1), (3, 65, 64, 1), (5, 1961, 64, 4),
                                    (1, 100000, 32, 128), (7, 31, 32, 2), (1, 2 ** 30 - 1, 64, 512),
                                    (1, 2 ** 30, 64, 512), (1, 2 ** 30 + 32, 64, 512),
                                    (1, 2 ** 30 + 32, 32, 1), (1, most, 64, 3), (1, most, 32, 512),
                                    (2 ** 24, 3, 64, 512)):
        out = subprocess.run([exe, *map(str, (segments, K, KS, splits))], check=True,
                             capture_output=True, text=True)
        assert int(out.stdout) == segments * K, (segments, K, KS, splits, out.stdout)


def test_token_counts_that_tiles_would_overflow_are_refused():
    from pwcnet_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(64)
    for M, text in ((2 ** 31 - 1, b"too large"), (2 ** 31 - 2 ** 16 + 1, b"too large"),
                    (2 ** 31 - 2 ** 16, b"null")):
        for layout in (0, 1):
            assert lib.pwc_linear_forward(None, p, None, None, p, layout, 1, M, 1, 1, 2 ** 31, 0, 0.1,
                                          2, None, 0, None) == 0
            assert text in lib.pwc_last_error(), lib.pwc_last_error()
            assert lib.pwc_gated_linear_backward(None, p, None, p, p, p, p, layout, 1, M, 1, 1,
                                                 2 ** 31, 0, 0.1, 2, None, 0, None) == 0
            assert text in lib.pwc_last_error(), lib.pwc_last_error()


# ------------------------------------------------------------------------------- the nodes
def test_statistics_of_the_norm_node_have_no_gradient():
    """A loss on them would get zeros: they do not ask for a gradient, compiled or not."""
    x = torch.empty(4, 8, device="meta", requires_grad=True)
    w = torch.empty(8, device="meta", requires_grad=True)

    def call(x, w):
        return torch.ops.pwcnet.layer_norm(x, w, None, 1e-5, -1)

    for f in (call, torch.compile(call, backend="aot_eager", fullgraph=True)):
        y, mean, rstd = f(x, w)
        assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
        for loss in (mean.sum(), rstd.sum()):
            with pytest.raises(RuntimeError, match="does not require grad"):
                loss.backward()
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and dw.shape == w.shape


# ------------------------------------------------------------------------------- workspaces
def test_norm_workspace_of_long_rows():
    """Partial sums of rows that no registers hold: as many as the kernel writes, a share of x."""
    from pwcnet_amd import _lib
    size = _lib.load().pwc_layer_norm_backward_workspace_size
    for M, C in ((1, 9000), (300, 9216), (20, 2 ** 20), (16384, 9216), (16384, 2 ** 20)):
        # [2][parts][C] in 32 bits, 32 rows at least to a part (and one part)
        assert 0 < size(1, 1, M, C, 2) <= 2 * (M // 32 + 1) * C * 4 + 255
    for B, P, C in ((1, 50, 300), (2, 5000, 2 ** 16), (16, 7168, 257)):
        assert 0 < size(0, B, P, C, 0) <= 2 * (B * P // 4096 + 1) * C * 4 + 255
    assert size(1, 1, 0, 9216, 2) == 0 and size(0, 3, 0, 300, 0) == 0


# ------------------------------------------------------------------------------- rotary
def test_rotary_refuses_what_it_has_no_gradient_for():
    """Frequencies and positions that ask for a gradient are refused, not left without one: by the
    function, by the node and compiled."""
    import pwcnet_amd as P
    f, a = P.rotary_frequencies((4,))
    x, at = torch.zeros(1, 5, 2, 8), torch.zeros(5, 1)
    ops = torch.ops.pwcnet
    for freq, places in ((f.clone().requires_grad_(True), at), (f, at.clone().requires_grad_(True))):
        with pytest.raises(ValueError, match="no gradient"):
            P.rotary(x, freq, a, places)
        meta = [t.detach().to("meta").requires_grad_(t.requires_grad) for t in (x, freq, a, places)]
        with pytest.raises(ValueError, match="no gradient"):
            ops.rotary(*meta, None, None, False, False)
        with pytest.raises(Exception, match="no gradient"):
            torch.compile(lambda *v: P.rotary(*v), backend="aot_eager")(*meta)
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP"):  # asks for none: as ever
        P.rotary(x, f.clone().requires_grad_(True), a, at)


def test_rotary_position_of_tokens_refuses_an_origin():
    """It was dropped; maps refuse it beside positions too."""
    import pwcnet_amd as P
    at = torch.zeros(5, 1, device="meta")
    m = P.RotaryPosition((4,), channel_dim=-1).to("meta")
    x = torch.empty(1, 5, 2, 8, device="meta")
    for places in (at, None):
        with pytest.raises(ValueError, match="origin"):
            m(x, places, origin=(3,))
    with pytest.raises(ValueError, match="origin"):
        m(x, origin=(0,))
