"""GPU: the feature operators called in other ways than eagerly on plain tensors, and at values and
sizes where a kernel's arithmetic could leave its formula."""
import math
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(*parts):
    return torch.Generator().manual_seed(zlib.crc32(repr(parts).encode()))


def _rand(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def u(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------- torch.jit.trace
@pytest.mark.filterwarnings("ignore")
def test_jit_trace_replays():
    """Traced operators, a block and rotary positions give the eager values and gradients on new
    inputs, with memory in between that an unfilled output would show."""
    import pwcnet_amd as P
    gen = _gen("trace")
    w, b = _rand(gen, 24, 16), _rand(gen, 24)
    n = _rand(gen, 16)
    calls = [lambda x: P.layer_norm(x, n, n), lambda x: P.linear(x, w, b, activation="gelu"),
             lambda x: P.gated_linear(x, w, b), P.RotaryPosition((4, 4)).to(DEV),
             P.FeatureBlock(16).to(DEV)]
    for call in calls:
        traced = torch.jit.trace(call, _rand(gen, 2, 16, 9, 11))
        for batch in (2, 3):
            x = _rand(gen, batch, 16, 9, 11).requires_grad_(True)
            want = call(x)
            g = _rand(gen, *want.shape)
            keep = torch.full((4, *want.shape), float("nan"), device=DEV)
            del keep
            got = traced(x)
            assert torch.equal(got, want)
            assert torch.equal(torch.autograd.grad(got, x, g)[0],
                               torch.autograd.grad(want, x, g)[0])


# ------------------------------------------------------------------------------- torch.func
@pytest.mark.filterwarnings("ignore")
def test_vmap_gives_each_samples_values():
    """vmap over samples, over weights and with gradients from outside: the eager results, sample by
    sample; torch.func.grad is refused, as for every node of the package."""
    import pwcnet_amd as P
    gen = _gen("vmap")
    x, w = _rand(gen, 3, 40, 16), _rand(gen, 3, 24, 16)
    inv, axis = P.rotary_frequencies((4, 4), device=DEV)
    at = torch.randint(0, 99, (40, 2), generator=gen).to(DEV)
    calls = [lambda x, w: P.layer_norm(x, channel_dim=-1),
             lambda x, w: P.linear(x, w, activation="gelu", channel_dim=-1),
             lambda x, w: P.gated_linear(x, w, channel_dim=-1),
             lambda x, w: P.rotary(x.view(1, 40, 1, 16), inv, axis, at)]
    for call in calls:
        want = torch.stack([call(x[k], w[k]) for k in range(3)])
        assert torch.equal(torch.vmap(call)(x, w), want)
        leaf = x.clone().requires_grad_(True)
        g = _rand(gen, *want.shape)
        got, = torch.autograd.grad(torch.vmap(call)(leaf, w), leaf, g)
        for k in range(3):
            one = x[k].clone().requires_grad_(True)
            assert torch.equal(got[k], torch.autograd.grad(call(one, w[k]), one, g[k])[0])
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v, w[0]).sum())(x[0])


# ------------------------------------------------------------------------------- long sums
def test_weight_gradient_of_an_image_past_2_30():
    """The weight gradient sums over an image's pixels: more than 2^30 of them, with the loads of the
    steps past the last outside."""
    from pwcnet_amd import features
    P_ = 2 ** 30 + 32
    x = torch.zeros(1, 2, P_, dtype=torch.bfloat16, device=DEV)
    dy = torch.zeros(1, 3, P_, dtype=torch.bfloat16, device=DEV)
    gen = _gen("long")
    at = torch.cat((torch.randint(0, P_, (4000,), generator=gen), torch.arange(P_ - 300, P_),
                    torch.arange(2 ** 30 - 70, 2 ** 30 + 3))).unique().to(DEV)
    x[0, :, at] = _rand(gen, 2, at.numel(), dtype=torch.bfloat16)
    dy[0, :, at] = _rand(gen, 3, at.numel(), dtype=torch.bfloat16)
    w = _rand(gen, 3, 2, dtype=torch.bfloat16)
    dw = features.linear_backward(x, w, None, dy, needs=(False, True, False))[1]
    a, b = dy[0, :, at].double(), x[0, :, at].double()
    ref = a @ b.t()
    # fp32 sums of the values that are there (zeros add nothing), then one rounding
    tol = at.numel() * 2.0 ** -24 * (a.abs() @ b.abs().t())
    assert ((dw.double() - ref).abs() <= tol + u(torch.bfloat16) * (ref.abs() + tol)).all()


# ------------------------------------------------------------------------------- activations
ACTS = ["none", "relu", "leaky_relu", "sigmoid", "tanh", "silu", "gelu", "gelu_tanh"]


def act64(z, name, slope=0.1):
    """act(z) in 64 bits"""
    if name == "relu":
        return z.clamp_min(0)
    if name == "leaky_relu":
        return torch.where(z > 0, z, slope * z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


# few tokens, tiles, parts of k, a map
PATHS = [((3, 64), 24, -1), ((200, 64), 72, -1), ((100, 2048), 520, -1), ((2, 64, 9, 8), 40, 1)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_activations_of_what_is_no_number(act, dtype):
    """Infinities and NaN, from the bias, through each activation on each path of the products: what
    the formula gives (-inf * 0 is no number there either)."""
    import pwcnet_amd as P
    for shape, O, dim in PATHS:
        x = _rand(_gen("no number", act), *shape, dtype=dtype)
        at = torch.tensor([math.inf, -math.inf, math.nan, 0.5, -2.0])
        b = at.repeat(O // 5 + 1)[:O].to(dtype).to(DEV)
        w = torch.zeros(O, x.shape[dim], dtype=dtype, device=DEV)
        want = act64(b.double(), act)
        for y in (P.linear(x, w, b, None, act, 0.1, dim),
                  P.gated_linear(x, torch.cat((w, w)), torch.cat((b, torch.ones_like(b))), act, 0.1,
                                 dim)):
            got = y.movedim(dim, -1).double()
            full = want.expand_as(got)
            whole = torch.isfinite(full)
            # (2^-20 for the activation in 32 bits, then the output's rounding)
            tol = u(dtype) * full.abs() + 2.0 ** -20
            assert ((got - full).abs() <= tol)[whole].all(), (shape, act)
            assert torch.equal(torch.isnan(got), torch.isnan(full)), (shape, act)
            inf = torch.isinf(full)
            assert torch.equal(got[inf], full[inf]), (shape, act)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gelu_of_far_negative_values(dtype):
    """gelu and its derivative where they fall below the type's step of 1: bounds relative to the
    value itself.

    The exponent of exp(-z^2 / 2) is rounded twice (2 z^2 / 2 2^-24 of the value: 2^-16 at -13), the
    tail's polynomial is off by 1.1e-5, a few roundings of 2^-24 follow: 2^-14.5 covers them.  Below
    the type's normal numbers half a step of the subnormal ones; and 32 bits' own (2^-149)."""
    import pwcnet_amd as P
    from pwcnet_amd import features
    z = torch.linspace(-13, -3, 520).to(dtype).to(DEV)
    zd = z.double()
    y = zd * torch.exp(torch.special.log_ndtr(zd))
    d = (torch.exp(torch.special.log_ndtr(zd))
         + zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi))
    floor = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2 + 2.0 ** -149
    rel = 2.0 ** -14.5
    for shape, O, dim in PATHS:
        if O < 520:
            b = z[::520 // O + 1]
            at = slice(None, None, 520 // O + 1)
        else:
            b, at = z, slice(None)
        x = _rand(_gen("far gelu"), *shape, dtype=dtype)
        w = torch.zeros(b.numel(), x.shape[dim], dtype=dtype, device=DEV)
        got = P.linear(x, w, b, activation="gelu", channel_dim=dim).movedim(dim, -1).double()
        assert ((got - y[at]).abs() <= (u(dtype) + rel) * y[at].abs() + floor).all(), shape
    # the bias gradient of one token is dz
    one = torch.ones(1, 520, dtype=dtype, device=DEV)
    w = torch.zeros(520, 8, dtype=dtype, device=DEV)
    db = features.linear_backward(one[:, :8].contiguous(), w, z, one, "gelu", channel_dim=-1)[2]
    assert ((db.double() - d).abs() <= (u(dtype) + rel) * d.abs() + floor).all()


# ------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("shape,dim", [((8, 32, 96, 112), 1), ((8, 20, 96, 101), 1), ((86016, 64), -1),
                                       ((3000, 2048), -1)])
def test_sums_over_blocks_in_pairs(shape, dim):
    """The bias gradient of 2^24 in the first row and 1 in every 64th, which additions one after the
    other to the large one would lose.

    At most 8 values of a block's own, 6 levels of its lanes, 2048 / 256 rounds and 8 levels of the
    blocks' sums follow one another, each off by at most 2^-24 of the total."""
    import pwcnet_amd as P
    dy = torch.zeros(shape, device=DEV)
    flat = dy.movedim(dim, -1)
    C, M = flat.shape[-1], flat.numel() // flat.shape[-1]
    n = torch.arange(M, device=DEV)
    one = torch.where(n % 64 == 0, 1.0, 0.0)
    one[0] = 2.0 ** 24
    flat.copy_(one.view(*flat.shape[:-1], 1).expand_as(flat))
    x = _rand(_gen("pairs", shape), *shape)
    b = torch.zeros(C, device=DEV, requires_grad=True)
    got, = torch.autograd.grad(P.layer_norm(x, None, b, channel_dim=dim), b, dy)
    want = one.double().sum()
    assert ((got.double() - want).abs() <= 30 * 2.0 ** -24 * want).all()


# ------------------------------------------------------------------------------- rotary
def test_rotary_refuses_negated_places():
    """Lazily negated positions and frequencies are refused, not read with the wrong sign."""
    import pwcnet_amd as P
    f, a = P.rotary_frequencies((4,), device=DEV)
    x = torch.zeros(1, 5, 2, 8, device=DEV)
    at = torch.ones(5, 1, device=DEV)
    neg_at = torch.conj(torch.complex(at, at)).imag
    neg_f = torch.conj(torch.complex(f, f)).imag
    assert neg_at.is_neg() and neg_f.is_neg()
    for freq, places in ((f, neg_at), (neg_f, at)):
        with pytest.raises(TypeError, match="negated"):
            P.rotary(x, freq, a, places)
    assert P.rotary(x, neg_f.resolve_neg(), a, neg_at.resolve_neg()).shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_activations_of_large_values(act, dtype):
    """Values up to the type's largest, whose squares and cubes are beyond 32 bits: the activation and
    its slope are finite wherever the formula's are.  (One rounding, 2^-20 for the functions.)"""
    import pwcnet_amd as P
    from pwcnet_amd import features
    most = torch.finfo(dtype).max
    at = [v for v in (30.0, 120.0, 6e4, 1e13, 1e19, 1e25, 3e38) if v <= most] + [most]
    z = torch.tensor([s * v for v in at for s in (1, -1)]).to(dtype).to(DEV)
    zd = z.double().requires_grad_(True)
    # (the cube and tanh's argument fit 64 bits)
    want = act64(zd, act)
    slope, = torch.autograd.grad(want.sum(), zd)
    if act in ("silu", "gelu", "gelu_tanh"):  # 0 * z of 64-bit autograd aside: 1 or 0 from 120 on
        slope = torch.where(zd.abs() >= 100, (zd > 0).double(), slope)
    want = want.detach()
    O = z.numel()
    w = torch.zeros(O, 8, dtype=dtype, device=DEV)
    for M in (1, 128):
        x = torch.ones(M, 8, dtype=dtype, device=DEV)
        y = P.linear(x, w, z, None, act, 0.1, -1).double()
        assert ((y - want).abs() <= u(dtype) * want.abs() + 2.0 ** -20).all(), (act, y)
        dy = torch.full((M, O), 1 / M, dtype=dtype, device=DEV)
        db = features.linear_backward(x, w, z, dy, act, 0.1, -1)[2].double()
        assert ((db - slope).abs() <= 2 * u(dtype) * slope.abs() + 2.0 ** -20).all(), (act, db)
