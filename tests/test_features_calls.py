"""CPU: ways of calling the feature operators other than eagerly on plain tensors (no call here
reaches a device), and what the entries ask for."""
import pytest
import torch


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
