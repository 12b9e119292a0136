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
