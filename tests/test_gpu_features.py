"""GPU: layer norm, rotary positions, linear and gated linear against their formulas in 64 bits.

Tolerances are bounds, element by element, from the kernels' arithmetic: one rounding of each output
(u = eps / 2 of its type), fp32 sums of n terms (n 2^-24 of the sum of their magnitudes), and, where
a backward pass multiplies with a dz kept in the storage type, u |dz| carried through that product.
The functions of the 64-bit side are written out here, with no operator of the package."""
import math
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "leaky_relu", "sigmoid", "tanh", "silu", "gelu", "gelu_tanh"]


def _gen(*parts):
    return torch.Generator().manual_seed(zlib.crc32(repr(parts).encode()))


def _rand(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def u(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):  # half a step of the subnormal numbers
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def _within(name, got, ref, tol):
    got, ref, tol = got.detach().double().cpu(), ref.detach().double().cpu(), tol.double().cpu()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    over = ((got - ref).abs() - tol)
    bad = ~(over <= 0)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst by "
                           f"{over[bad].max().item():.3g} at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {ref[bad][0].item()}, "
                           f"allowed {tol[bad][0].item():.3g}")


def act64(z, name, slope=0.1):
    """(act(z), act'(z)) in 64 bits"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "leaky_relu":
        return torch.where(z > 0, z, slope * z), torch.where(z > 0, 1.0, slope).double()
    if name == "sigmoid":
        p = torch.sigmoid(z)
        return p, p * (1 - p)
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    p = torch.sigmoid(2 * a)
    return z * p, p + 2 * z * p * (1 - p) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)


def _tok(t, is_map):
    """[B, C, *spatial] -> [M, C] (tokens unchanged, leading dimensions joined)"""
    return t.movedim(1, -1).reshape(-1, t.shape[1]) if is_map else t.reshape(-1, t.shape[-1])


class Product64:
    """linear / gated linear in 64 bits on [M, K], with the bounds of what the kernels return."""

    def __init__(self, x, w, b, act, slope, gated, dtype, res=None):
        self.x, self.w, self.gated, self.u = x.double(), w.double(), gated, u(dtype)
        self.kept = u(dtype)  # what dz loses where the backward keeps it
        self.floor = _floor(dtype)
        self.act = act
        K = x.shape[1]
        z = self.x @ self.w.t() + (b.double() if b is not None else 0)
        # fp32 sum of K products and the bias
        self.ez = (K + 4) * F32 * (self.x.abs() @ self.w.abs().t()
                                   + (b.double().abs() if b is not None else 0))
        if gated:
            n = w.shape[0] // 2
            self.zg, self.zu, self.eg, self.eu = z[:, :n], z[:, n:], self.ez[:, :n], self.ez[:, n:]
            self.f, self.df = act64(self.zg, act, slope)
            self.y = self.f * self.zu
            # |act'| <= 1.13 everywhere; the activation itself within 2^-20 of its magnitude
            ef = 1.2 * self.eg + 2.0 ** -20 * (self.f.abs() + self.zg.abs() * 2.0 ** -3)
            self.ef = ef
            err = ef * self.zu.abs() + self.f.abs() * self.eu + ef * self.eu
        else:
            self.zg, self.eg = z, self.ez
            self.f, self.df = act64(z, act, slope)
            self.y = self.f + (res.double() if res is not None else 0)
            self.ef = 1.2 * self.ez + 2.0 ** -20 * (self.f.abs() + z.abs() * 2.0 ** -3)
            err = self.ef + (F32 * (self.f.abs() + res.double().abs()) if res is not None else 0)
        self.tol_y = err + self.u * (self.y.abs() + err) + self.floor

    def backward(self, dy):
        dy = dy.double()
        # |act''| <= 1.2; at a kink the other branch is as good where z is within its error
        edf = 1.2 * self.eg + 2.0 ** -20
        if self.act in ("relu", "leaky_relu"):
            edf = torch.where(self.zg.abs() <= self.eg, 1.0, 2.0 ** -23).double()
        if self.act == "none":
            edf = torch.zeros_like(self.zg)
        if self.gated:
            dz = torch.cat((dy * self.zu * self.df, dy * self.f), 1)
            e = torch.cat((dy.abs() * (self.zu.abs() * edf + self.eu * (self.df.abs() + edf)),
                           dy.abs() * self.ef), 1)
        else:
            dz = dy * self.df
            e = dy.abs() * edf
        if self.gated or self.act != "none":  # kept in the storage type
            e = e + 3 * F32 * dz.abs()
            e = e + self.kept * (dz.abs() + e) + self.floor
        M, rows = dz.shape
        a = dz.abs() + e
        out = {}
        for name, v, err in (
                ("dx", dz @ self.w, e @ self.w.abs() + (rows + 2) * F32 * (a @ self.w.abs())),
                ("dw", dz.t() @ self.x,
                 e.t() @ self.x.abs() + (M + 300) * F32 * (a.t() @ self.x.abs())),
                ("db", dz.sum(0), e.sum(0) + (M + 300) * F32 * a.sum(0))):
            out[name] = (v, err + self.u * (v.abs() + err) + self.floor)
        return out


def _product_case(is_map, dims, K, O, dtype, act, bias, residual, gated, seed=0):
    gen = _gen(is_map, dims, K, O, str(dtype), act, bias, residual, gated, seed)
    shape = (dims[0], K, *dims[1:]) if is_map else (*dims, K)
    oshape = (dims[0], O, *dims[1:]) if is_map else (*dims, O)
    rows = 2 * O if gated else O
    x = _rand(gen, *shape, dtype=dtype, shift=0.3)
    w = _rand(gen, rows, K, dtype=dtype, scale=K ** -0.5)
    b = _rand(gen, rows, dtype=dtype, scale=0.5) if bias else None
    r = _rand(gen, *oshape, dtype=dtype) if residual else None
    g = _rand(gen, *oshape, dtype=dtype)
    return x, w, b, r, g


def _check_product(x, w, b, r, g, act, gated, channel_dim):
    import pwcnet_amd as P
    is_map = channel_dim == 1
    dtype = x.dtype
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    if gated:
        y = P.gated_linear(x, w, b, act, 0.2, channel_dim)
    else:
        y = P.linear(x, w, b, r, act, 0.2, channel_dim)
    grads = torch.autograd.grad(y, leaves, g)
    with torch.no_grad():
        # without a graph: the same values
        again = (P.gated_linear(x, w, b, act, 0.2, channel_dim) if gated
                 else P.linear(x, w, b, r, act, 0.2, channel_dim))
        assert torch.equal(again, y)
        ref = Product64(_tok(x, is_map), w, b, act, 0.2, gated, dtype,
                        _tok(r, is_map) if r is not None else None)
        _within("y", _tok(y, is_map), ref.y, ref.tol_y)
        back = ref.backward(_tok(g, is_map))
        _within("dx", _tok(grads[0], is_map), *back["dx"])
        _within("dw", grads[1], *back["dw"])
        if b is not None:
            _within("db", grads[2], *back["db"])
        if r is not None:
            assert torch.equal(grads[-1], g)


TOKENS = [((1,), 1, 1), ((1,), 8, 8), ((5,), 33, 17), ((2, 3), 64, 130), ((130,), 257, 129),
          ((257,), 64, 64), ((64,), 128, 304), ((300,), 520, 96), ((3,), 1000, 72), ((129,), 24, 1)]
MAPS = [((1, 1, 1), 1, 1), ((2, 3, 5), 4, 6), ((3, 7, 9), 33, 17), ((2, 16, 16), 32, 64),
        ((1, 37, 53), 96, 40), ((2, 12, 14), 136, 72), ((5, 1, 3), 8, 8), ((1, 24, 28), 200, 130)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", range(len(TOKENS)))
def test_linear_tokens(n, dtype):
    dims, K, O = TOKENS[n]
    act = ACTS[n % len(ACTS)]
    case = _product_case(False, dims, K, O, dtype, act, n % 3 != 1, n % 2 == 0, False)
    _check_product(*case, act, False, -1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", range(len(MAPS)))
def test_linear_map(n, dtype):
    dims, K, O = MAPS[n]
    act = ACTS[(n + 2) % len(ACTS)]
    case = _product_case(True, dims, K, O, dtype, act, n % 3 != 1, n % 2 == 1, False)
    _check_product(*case, act, False, 1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", range(len(TOKENS)))
def test_gated_tokens(n, dtype):
    dims, K, O = TOKENS[n]
    act = ACTS[(n + 5) % len(ACTS)]
    case = _product_case(False, dims, K, O, dtype, act, n % 3 != 2, False, True)
    case = (*case[:3], None, case[4])
    _check_product(*case, act, True, -1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", range(len(MAPS)))
def test_gated_map(n, dtype):
    dims, K, O = MAPS[n]
    act = ACTS[(n + 4) % len(ACTS)]
    case = _product_case(True, dims, K, O, dtype, act, n % 3 != 2, False, True)
    _check_product(*case, act, True, 1)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_every_activation(act, gated, dtype):
    case = _product_case(False, (70,), 40, 48, dtype, act, True, not gated, gated)
    _check_product(*case, act, gated, -1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 33])
def test_few_tokens(tokens, dtype):
    """Single tokens and small batches of them against long rows."""
    for K, O, gated in ((1024, 520, False), (1536, 200, True), (777, 65, False), (129, 50, True)):
        case = _product_case(False, (tokens,), K, O, dtype, "silu", True, not gated, gated)
        _check_product(*case, "silu", gated, -1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("is_map,dims,K,O,gated", [
    (False, (1,), 512, 96, False), (False, (7,), 264, 130, True), (False, (40,), 1000, 65, True),
    (False, (3440,), 176, 8, True), (False, (777,), 65, 33, False), (False, (301,), 511, 509, False),
    (False, (150,), 773, 257, True), (True, (7, 3, 2), 1, 40, False),
    (True, (3, 24, 28), 32, 48, True), (True, (2, 37, 53), 33, 17, True)])
def test_small_gradients_keep_their_bits(is_map, dims, K, O, gated, dtype):
    """In small 16-bit calls dz is kept in two parts, u^2 off instead of u (the second part of a
    16-bit value is at most u of it and rounded itself; fp16's is off by the subnormal step too)."""
    import pwcnet_amd as P
    x, w, b, _, g = _product_case(is_map, dims, K, O, dtype, "silu", True, False, gated)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = (P.gated_linear if gated else P.linear)(x, w, b, activation="silu",
                                               channel_dim=1 if is_map else -1)
    grads = torch.autograd.grad(y, leaves, g)
    with torch.no_grad():
        ref = Product64(_tok(x, is_map), w, b, "silu", 0.1, gated, dtype)
        ref.kept = u(dtype) ** 2
        back = ref.backward(_tok(g, is_map))
        _within("dx", _tok(grads[0], is_map), *back["dx"])
        _within("dw", grads[1], *back["dw"])


def test_small_gradients_beyond_the_type():
    """A dz that rounds to infinity gives infinite gradients, no NaN."""
    import pwcnet_amd as P
    for tokens in (3, 70):
        x = torch.full((tokens, 32), 4.0, dtype=torch.float16, device=DEV, requires_grad=True)
        w = torch.full((48, 32), 0.25, dtype=torch.float16, device=DEV, requires_grad=True)
        y = P.gated_linear(x, w, None, "silu", channel_dim=-1)
        dx, dw = torch.autograd.grad(y, (x, w), torch.full_like(y, 65504.0))
        assert bool(torch.isposinf(dx).all()) and bool(torch.isposinf(dw).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens", [33, 48, 64, 100, 255, 513])
def test_some_tokens(tokens, dtype):
    """Too few tokens to fill the card: long rows are summed in parts, whatever follows."""
    for K, O, gated, act in ((2048, 520, False, "gelu"), (1536, 200, True, "silu"),
                             (2055, 67, False, "none"), (1032, 51, True, "gelu_tanh"),
                             (2053, 1021, False, "silu"), (1029, 2047, True, "silu")):
        case = _product_case(False, (tokens,), K, O, dtype, act, True, not gated, gated)
        _check_product(*case, act, gated, -1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_few_tokens_long_gradients(dtype):
    """dx of few tokens over many output channels is summed in parts."""
    for tokens, K, O, gated in ((1, 264, 2100, False), (7, 96, 1500, True), (64, 65, 1031, False),
                                (65, 200, 1024, True)):
        for act in ("none", "gelu"):
            case = _product_case(False, (tokens,), K, O, dtype, act, True, False, gated)
            _check_product(*case, act, gated, -1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_steps(dtype):
    """Long sums on both sides of the weight gradient's split, several tiles each way."""
    for is_map, dims, K, O in ((False, (3000,), 200, 264), (True, (3, 40, 50), 72, 136),
                               (True, (2, 31, 33), 160, 300)):
        for gated in (False, True):
            case = _product_case(is_map, dims, K, O, dtype, "gelu", True, not gated, gated)
            _check_product(*case, "gelu", gated, 1 if is_map else -1)


@pytest.mark.parametrize("dtype,is_map,dims,K,O,gated,act", [
    (torch.bfloat16, False, (3001,), 517, 1021, False, "gelu"),
    (torch.float16, False, (3001,), 520, 1021, False, "none"),
    (torch.bfloat16, False, (2999,), 521, 1024, False, "none"),
    (torch.float16, False, (4093,), 259, 517, True, "silu"),
    (torch.bfloat16, True, (4, 61, 67), 131, 259, True, "silu"),
    (torch.float16, True, (5, 61, 67), 136, 392, False, "none"),
    (torch.bfloat16, True, (4, 62, 68), 133, 517, False, "gelu_tanh"),
    (torch.float32, False, (4099,), 1021, 1019, False, "tanh")])
def test_large_rows_at_odd_places(dtype, is_map, dims, K, O, gated, act):
    """Large products whose rows are laid out at 16-byte places first."""
    case = _product_case(is_map, dims, K, O, dtype, act, True, not gated, gated)
    _check_product(*case, act, gated, 1 if is_map else -1)


def test_large_rows_with_a_distance():
    """A slice of a wider buffer (odd distance, odd start) gives its copy's values; what stands
    between the rows is not read into the sums."""
    import pwcnet_amd as P
    gen = _gen("distance")
    wide = torch.full((4100, 1051), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[2:4098, 3:1027] = _rand(gen, 4096, 1024, dtype=torch.bfloat16)
    x = wide[2:4098, 3:1027]
    w, g = (_rand(gen, 512, 1024, dtype=torch.bfloat16, scale=1 / 32),
            _rand(gen, 4096, 512, dtype=torch.bfloat16))
    want = None
    for v in (x.contiguous(), x):
        v = v.detach().requires_grad_(True)
        u = w.clone().requires_grad_(True)
        y = P.linear(v, u, activation="silu", channel_dim=-1)
        got = [y.detach(), *torch.autograd.grad(y, (v, u), g)]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_large_tiles(dtype):
    """Enough rows and columns for the largest tiles, one short of and one past a tile."""
    for M, K, O, gated in ((2049, 264, 1288, False), (2047, 128, 640, True), (1024, 512, 1024, False)):
        case = _product_case(False, (M,), K, O, dtype, "silu", True, False, gated)
        _check_product(*case, "silu", gated, -1)


def test_products_do_not_mix_rows():
    """What stands outside a row or a token -- neighbours that are not numbers -- stays outside."""
    import pwcnet_amd as P
    for dtype in DTYPES:
        gen = _gen("mix", str(dtype))
        for M, K, O in ((5, 37, 21), (40, 64, 72), (1, 40, 24)):
            wide = torch.full((M + 2, K + 8), float("nan"), dtype=dtype, device=DEV)
            wide[1:-1, :K] = _rand(gen, M, K, dtype=dtype)
            x = wide[1:-1, :K]
            w, b = _rand(gen, O, K, dtype=dtype), _rand(gen, O, dtype=dtype)
            assert torch.equal(P.linear(x, w, b, channel_dim=-1),
                               P.linear(x.contiguous(), w, b, channel_dim=-1))
            g = _rand(gen, M, O, dtype=dtype)
            xs = x.clone().requires_grad_(True)
            w.requires_grad_(True)
            a = torch.autograd.grad(P.linear(xs, w, b, activation="silu", channel_dim=-1),
                                    (xs, w), g)
            xw = wide.requires_grad_(True)[1:-1, :K]
            c = torch.autograd.grad(P.linear(xw, w, b, activation="silu", channel_dim=-1),
                                    (wide, w), g)
            assert torch.equal(a[1], c[1]) and torch.equal(a[0], c[0][1:-1, :K])
            w.requires_grad_(False)
        # images at a distance
        buf = torch.full((3, 20, 6, 7), float("nan"), dtype=dtype, device=DEV)
        buf[:, 3:15] = _rand(gen, 3, 12, 6, 7, dtype=dtype)
        w = _rand(gen, 10, 12, dtype=dtype)
        assert torch.equal(P.linear(buf[:, 3:15], w), P.linear(buf[:, 3:15].contiguous(), w))
        # a token that is not a number leaves the others
        x = _rand(gen, 9, 48, dtype=dtype)
        y = P.linear(x, w.new_ones(8, 48), channel_dim=-1)
        x[4, 5] = float("inf")
        x[6, 7] = float("nan")
        z = P.linear(x, w.new_ones(8, 48), channel_dim=-1)
        keep = [0, 1, 2, 3, 5, 7, 8]
        assert torch.equal(y[keep], z[keep])
        assert torch.isinf(z[4]).all() and torch.isnan(z[6]).all()


def test_product_strides_and_orders():
    """Transposed, broadcast, sliced and channels-last operands give the values of their copies."""
    import pwcnet_amd as P
    gen = _gen("strides")
    for dtype in DTYPES:
        w, b = _rand(gen, 24, 40, dtype=dtype), _rand(gen, 24, dtype=dtype)
        cases = [(_rand(gen, 40, 30, dtype=dtype).t(), -1),
                 (_rand(gen, 1, 40, dtype=dtype).expand(7, 40), -1),
                 (_rand(gen, 6, 5, 40, dtype=dtype).transpose(0, 1), -1),
                 (_rand(gen, 10, 5, 40, dtype=dtype)[::2], -1),
                 (_rand(gen, 10, 41, dtype=dtype)[:, 1:], -1),
                 (_rand(gen, 10, 80, dtype=dtype)[:, ::2], -1),
                 (_rand(gen, 2, 40, 6, 7, dtype=dtype).to(memory_format=torch.channels_last), 1),
                 (_rand(gen, 2, 40, 6, 7, dtype=dtype).transpose(2, 3), 1),
                 (_rand(gen, 1, 40, 6, 7, dtype=dtype).expand(3, 40, 6, 7), 1),
                 (_rand(gen, 2, 45, 5, 7, dtype=dtype)[:, 5:], 1),
                 (_rand(gen, 4, 40, 9, dtype=dtype)[1::2], 1),
                 (_rand(gen, 3, 40, dtype=dtype), 1)]
        for x, ch in cases:
            got = P.linear(x, w, b, activation="gelu", channel_dim=ch)
            assert torch.equal(got, P.linear(x.contiguous().clone(), w, b, activation="gelu",
                                             channel_dim=ch))
            shape = list(x.shape)
            shape[ch] = 24
            assert list(got.shape) == shape
        x = _rand(gen, 7, 40, dtype=dtype)
        wt = _rand(gen, 40, 24, dtype=dtype).t()
        assert torch.equal(P.linear(x, wt, b, channel_dim=-1),
                           P.linear(x, wt.contiguous(), b, channel_dim=-1))
        res = _rand(gen, 1, 24, dtype=dtype).expand(7, 24)
        assert torch.equal(P.linear(x, w, b, res, channel_dim=-1),
                           P.linear(x, w, b, res.contiguous(), channel_dim=-1))


def test_product_gradients_against_differences():
    """fp32 gradients against central differences of the 64-bit forward formula."""
    import pwcnet_amd as P
    gen = _gen("differences")
    x, w, b = (_rand(gen, 6, 9), _rand(gen, 14, 9, scale=0.3), _rand(gen, 14))
    g = _rand(gen, 6, 7)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(P.gated_linear(x, w, b, "gelu_tanh", channel_dim=-1), (x, w, b), g)

    def loss(x, w, b):
        z = x @ w.t() + b
        return float((act64(z[:, :7], "gelu_tanh")[0] * z[:, 7:] * g.double()).sum())

    leaves = [t.detach().double() for t in (x, w, b)]
    h = 1e-4  # differences: h^2 f''' / 6 ~ 1e-8 of the gradient's size
    for n, grad in enumerate(grads):
        flat = leaves[n].view(-1)
        for at in range(0, flat.numel(), 5):
            keep = flat[at].item()
            flat[at] = keep + h
            up = loss(*leaves)
            flat[at] = keep - h
            down = loss(*leaves)
            flat[at] = keep
            assert abs((up - down) / (2 * h) - grad.view(-1)[at].item()) < 2e-5


# ------------------------------------------------------------------------------- layer norm
def _norm64(x, w, b, eps, dtype, dy):
    """(name -> (value, bound)) for x [M, C] in 64 bits; see the kernels' passes."""
    x, dy = x.double(), dy.double()
    M, C = x.shape
    w = w.double() if w is not None else torch.ones(C, dtype=torch.float64, device=DEV)
    b = b.double() if b is not None else torch.zeros(C, dtype=torch.float64, device=DEV)
    mu = x.mean(1, keepdim=True)
    d = x - mu
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    xh = d * r
    y = xh * w + b
    em = (C + 1) * F32 * x.abs().mean(1, keepdim=True)      # of the mean
    er = (C + 8) * F32 + (r * em) ** 2                       # of r, relative
    exh = r * em + xh.abs() * (er + 2 * F32)
    uu, fl = u(dtype), _floor(dtype)
    ey = w.abs() * exh + 3 * F32 * ((xh * w).abs() + b.abs())
    h = dy * w
    m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    dx = r * (h - m1 - xh * m2)
    e2 = (C + 3) * F32 * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * exh).mean(1, keepdim=True)
    edx = er * dx.abs() + r * (4 * F32 * h.abs() + (C + 4) * F32 * h.abs().mean(1, keepdim=True)
                               + exh * (m2.abs() + e2) + xh.abs() * (e2 + 4 * F32 * m2.abs()))
    edw = (dy.abs() * exh).sum(0) + (M + 40) * F32 * (dy * xh).abs().sum(0)
    edb = (M + 40) * F32 * dy.abs().sum(0)
    out = {}
    for name, v, e in (("y", y, ey), ("dx", dx, edx), ("dw", (dy * xh).sum(0), edw),
                       ("db", dy.sum(0), edb)):
        out[name] = (v, e + uu * (v.abs() + e) + fl)
    return out


def _check_norm(x, w, b, dy, channel_dim, eps=1e-5):
    import pwcnet_amd as P
    is_map = channel_dim == 1
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = P.layer_norm(x, w, b, eps, channel_dim)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(P.layer_norm(x, w, b, eps, channel_dim), y)
        ref = _norm64(_tok(x, is_map), w, b, eps, x.dtype, _tok(dy, is_map))
        _within("y", _tok(y, is_map), *ref["y"])
        _within("dx", _tok(grads[0], is_map), *ref["dx"])
        if w is not None:
            _within("dw", grads[1], *ref["dw"])
        if b is not None:
            _within("db", grads[-1], *ref["db"])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("C", [1, 2, 3, 7, 8, 16, 32, 33, 96, 128, 129, 200, 1000, 1024, 1025,
                               2048, 2500, 4097, 8192, 8193, 9000])
def test_layer_norm_tokens(C, dtype):
    gen = _gen("norm", C, str(dtype))
    for M in (1, 5, 300):
        x = _rand(gen, M, C, dtype=dtype, shift=0.5)
        w, b = _rand(gen, C, dtype=dtype, shift=1), _rand(gen, C, dtype=dtype)
        _check_norm(x, w if M != 5 else None, b if M != 1 else None,
                    _rand(gen, M, C, dtype=dtype), -1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("C", [1, 2, 3, 16, 17, 32, 64, 65, 96, 128, 129, 192, 256, 257, 300, 513,
                               1000])
def test_layer_norm_map(C, dtype):
    gen = _gen("norm map", C, str(dtype))
    for dims in ((1, 1, 1), (2, 3, 5), (3, 16, 16), (2, 7, 19), (1, 8, 8)):
        x = _rand(gen, dims[0], C, *dims[1:], dtype=dtype, shift=-0.5)
        w, b = _rand(gen, C, dtype=dtype, shift=1), _rand(gen, C, dtype=dtype)
        _check_norm(x, w if dims[0] != 2 else None, b if dims[0] != 1 else None,
                    _rand(gen, dims[0], C, *dims[1:], dtype=dtype), 1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layer_norm_many_rows(dtype):
    """More rows than the blocks that stay: each takes several turns."""
    gen = _gen("norm rows", str(dtype))
    for M, C in ((70000, 8), (9001, 72), (5003, 1032), (301, 9216)):
        x = _rand(gen, M, C, dtype=dtype, shift=0.5)
        _check_norm(x, _rand(gen, C, dtype=dtype), _rand(gen, C, dtype=dtype),
                    _rand(gen, M, C, dtype=dtype), -1)
    for B, C, H, W in ((8, 20, 96, 101), (9, 70, 88, 88), (3, 270, 48, 57)):
        x = _rand(gen, B, C, H, W, dtype=dtype, shift=0.5)
        _check_norm(x, _rand(gen, C, dtype=dtype), _rand(gen, C, dtype=dtype),
                    _rand(gen, B, C, H, W, dtype=dtype), 1)


def test_layer_norm_far_mean():
    """A mean 1000 times the spread costs the digits it must, and no more: sum of x - mean."""
    import pwcnet_amd as P
    gen = _gen("far")
    x = _rand(gen, 40, 512, shift=1000.0)
    ref = _norm64(x, None, None, 1e-5, torch.float32, x)
    _within("y", P.layer_norm(x, channel_dim=-1), *ref["y"])
    # a plain sum of squares would be off by 1e6 * 2^-24 * r here
    assert (P.layer_norm(x, channel_dim=-1).double() - ref["y"][0]).abs().max() < 2e-4
    x = _rand(gen, 2, 48, 9, 9, shift=1000.0)
    ref = _norm64(_tok(x, True), None, None, 1e-5, torch.float32, _tok(x, True))
    assert (_tok(P.layer_norm(x), True).double() - ref["y"][0]).abs().max() < 2e-4


def test_layer_norm_constant_rows_and_neighbours():
    """A row of equal values is its bias; rows that are not numbers leave the others; strided rows
    with such neighbours give the values of their copies."""
    import pwcnet_amd as P
    gen = _gen("constant")
    for dtype in DTYPES:
        for C in (5, 64, 300):
            b = _rand(gen, C, dtype=dtype)
            x = torch.full((6, C), 3.0, dtype=dtype, device=DEV)
            assert torch.equal(P.layer_norm(x, None, b, channel_dim=-1), b.expand(6, C))
            x = _rand(gen, 6, C, dtype=dtype)
            y = P.layer_norm(x, None, b, channel_dim=-1)
            x[2, C // 2] = float("nan")
            x[4, 0] = float("inf")
            z = P.layer_norm(x, None, b, channel_dim=-1)
            assert torch.equal(y[[0, 1, 3, 5]], z[[0, 1, 3, 5]])
            assert torch.isnan(z[2]).all() and torch.isnan(z[4]).all()
            wide = torch.full((8, C + 3), float("nan"), dtype=dtype, device=DEV)
            wide[1:7, 1:C + 1] = _rand(gen, 6, C, dtype=dtype)
            v = wide[1:7, 1:C + 1]
            assert torch.equal(P.layer_norm(v, channel_dim=-1),
                               P.layer_norm(v.contiguous(), channel_dim=-1))
        buf = torch.full((2, 12, 5, 5), float("nan"), dtype=dtype, device=DEV)
        buf[:, 2:9] = _rand(gen, 2, 7, 5, 5, dtype=dtype)
        assert torch.equal(P.layer_norm(buf[:, 2:9]), P.layer_norm(buf[:, 2:9].contiguous()))


# ------------------------------------------------------------------------------- rotary
def _rotary64(x, inv_freq, axis, at, interleaved, sign=1.0):
    """x [B, N, H, D], at [B or 1, N, A]: (value, bound)"""
    R = inv_freq.numel()
    a = at.double()[..., axis.long()] * inv_freq
    c, s = torch.cos(a)[:, :, None], sign * torch.sin(a)[:, :, None]
    v = x.double()
    y, mag = v.clone(), torch.zeros_like(v)
    i = slice(0, 2 * R, 2) if interleaved else slice(0, R)
    j = slice(1, 2 * R, 2) if interleaved else slice(R, 2 * R)
    y[..., i] = v[..., i] * c - v[..., j] * s
    y[..., j] = v[..., i] * s + v[..., j] * c
    mag[..., i] = mag[..., j] = v[..., i].abs() + v[..., j].abs()
    # angle rounded to 2^-25 of a turn, sine and cosine to two steps, the sum to two; and the
    # angle in 64 bits: the product here (2^-53 of it), there 1 / 2 pi, its product with the
    # frequency and the product with the place (2^-53 each) -- 2^33 radians make 2^-18 of that
    far = torch.zeros_like(v)
    far[..., i] = far[..., j] = 4 * 2.0 ** -53 * a.abs()[:, :, None]
    tol = (2.0 ** -21 + far) * mag
    tol = tol + u(x.dtype) * (y.abs() + tol) + torch.where(mag > 0, _floor(x.dtype), 0.0)
    tol[..., 2 * R:] = 0
    return y, tol


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,H,D,sections", [
    (1, 1, 1, 2, (1,)), (2, 5, 3, 16, (8,)), (3, 17, 2, 32, (4, 12)), (1, 70, 5, 64, (8, 12, 12)),
    (2, 9, 4, 80, (16, 8)), (4, 1, 32, 128, (16, 24, 24)), (2, 33, 2, 7, (1, 1)),
    (1, 300, 24, 128, (64,)), (2, 6, 1, 24, (2, 3, 4, 3)), (2, 40, 3, 96, (8, 16, 8))])
def test_rotary_tokens(B, N, H, D, sections, interleaved, dtype):
    import pwcnet_amd as P
    gen = _gen("rotary", B, N, H, D, sections, interleaved, str(dtype))
    inv_freq, axis = P.rotary_frequencies(sections, device=DEV)
    x = _rand(gen, B, N, H, D, dtype=dtype).requires_grad_(True)
    g = _rand(gen, B, N, H, D, dtype=dtype)
    for kind in (torch.int64, torch.int32, torch.float32):
        at = torch.randint(-500, 100000, (B if kind != torch.int32 else 1, N, len(sections)),
                           generator=gen).to(DEV)
        if kind == torch.float32:
            at = at / 64  # exact, between whole places
        at = at.to(kind)
        y = P.rotary(x, inv_freq, axis, at, interleaved=interleaved)
        _within("y", y, *_rotary64(x, inv_freq, axis, at, interleaved))
        dx, = torch.autograd.grad(y, x, g)
        _within("dx", dx, *_rotary64(g, inv_freq, axis, at, interleaved, -1.0))
    with torch.no_grad():  # positions of one image for all
        assert torch.equal(P.rotary(x, inv_freq, axis, at[0], interleaved=interleaved),
                           P.rotary(x, inv_freq, axis, at[:1].expand(B, -1, -1),
                                    interleaved=interleaved))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,heads,C,H,W,sections", [
    (1, 1, 2, 1, 1, (1, 0)), (2, 1, 32, 6, 7, (8, 8)), (3, 2, 40, 8, 16, (4, 6)),
    (16, 1, 32, 12, 32, (0, 8, 8)), (2, 4, 96, 5, 9, (2, 3, 4)), (5, 1, 9, 3, 8, (2, 2))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_map(B, heads, C, H, W, sections, interleaved, dtype):
    import pwcnet_amd as P
    gen = _gen("rotary map", B, heads, C, H, W, sections, interleaved, str(dtype))
    m = P.RotaryPosition(sections, heads=heads, interleaved=interleaved).to(DEV)
    x = _rand(gen, B, C, H, W, dtype=dtype).requires_grad_(True)
    g = _rand(gen, B, C, H, W, dtype=dtype)
    origin = [7, 100, 3000][:len(sections)]
    at = torch.stack(torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij"), -1)
    at = at.reshape(1, H * W, 2).to(DEV) + torch.tensor(origin[-2:], device=DEV)
    if len(sections) == 3:
        at = torch.cat((torch.full_like(at[..., :1], origin[0]), at), -1)
    y = m(x, origin=origin)
    assert y.shape == x.shape and y.is_contiguous()

    def heads_last(t):
        return t.reshape(B, heads, C // heads, H * W).permute(0, 3, 1, 2)

    _within("y", heads_last(y), *_rotary64(heads_last(x), m.inv_freq, m.axis, at, interleaved))
    dx, = torch.autograd.grad(y, x, g)
    _within("dx", heads_last(dx), *_rotary64(heads_last(g), m.inv_freq, m.axis, at, interleaved,
                                             -1.0))
    with torch.no_grad():
        assert torch.equal(m(x, positions=at), y)


def test_rotary_strides_and_rest():
    """Head-first tokens, slices of a joint projection and odd strides give the values of their
    copies; what passes is copied bit by bit, also where it is no number."""
    import pwcnet_amd as P
    gen = _gen("rotary strides")
    inv_freq, axis = P.rotary_frequencies((4, 4, 8), device=DEV)
    for dtype in DTYPES:
        at = torch.randint(0, 999, (2, 11, 3), generator=gen).to(DEV)
        joint = _rand(gen, 2, 11, (4 + 2) * 40, dtype=dtype)
        views = [joint[..., :160].view(2, 11, 4, 40), joint[..., 160:200].view(2, 11, 1, 40),
                 _rand(gen, 2, 4, 11, 40, dtype=dtype).transpose(1, 2),
                 _rand(gen, 2, 4, 40, 11, dtype=dtype).permute(0, 3, 1, 2),
                 _rand(gen, 2, 11, 4, 80, dtype=dtype)[..., ::2],
                 _rand(gen, 1, 11, 4, 40, dtype=dtype).expand(2, 11, 4, 40),
                 _rand(gen, 2, 11, 4, 41, dtype=dtype)[..., 1:]]
        for x in views:
            ref = P.rotary(x.contiguous(), inv_freq, axis, at)
            assert torch.equal(P.rotary(x, inv_freq, axis, at), ref)
            assert torch.equal(P.rotary(x, inv_freq, axis, at.transpose(0, 2).contiguous()
                                        .transpose(0, 2)), ref)
        x = _rand(gen, 2, 11, 4, 40, dtype=dtype)
        x[..., 32:] = float("nan")
        x[0, ..., 35] = float("inf")
        for v in (x, x.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)):
            y = P.rotary(v, inv_freq, axis, at)
            assert torch.isfinite(y[..., :32]).all()
            assert torch.equal(y[..., 32:].nan_to_num(7.0), x[..., 32:].nan_to_num(7.0))


def test_rotary_far_positions():
    """Places past 2^31, and a turn followed by its inverse."""
    import pwcnet_amd as P
    from pwcnet_amd import features
    gen = _gen("far places")
    inv_freq, axis = P.rotary_frequencies((16,), device=DEV)
    x = _rand(gen, 1, 6, 2, 32)
    at = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 + 5, 2 ** 33 + 7, -(2 ** 32) - 3]).view(1, 6, 1)
    y = P.rotary(x, inv_freq, axis, at.to(DEV))
    _within("y", y, *_rotary64(x, inv_freq, axis, at.to(DEV), False))
    back = features.rotary_forward(y, inv_freq, axis, at.to(DEV), inverse=True)
    # both turns use the same rounded angle
    assert (back - x).abs().max() < 2.0 ** -19 * x.abs().max()
    z = P.rotary(x, inv_freq, axis, grid=(6,), origin=(2 ** 33,))
    _within("z", z, *_rotary64(x, inv_freq, axis, (torch.arange(6, device=DEV) + 2 ** 33)
                               .view(1, 6, 1), False))


# ------------------------------------------------------------------------------- all of them
def test_empty_batches():
    import pwcnet_amd as P
    for dtype in DTYPES:
        w = torch.ones(6, 4, dtype=dtype, device=DEV, requires_grad=True)
        b = torch.ones(6, dtype=dtype, device=DEV, requires_grad=True)
        n = torch.ones(4, dtype=dtype, device=DEV, requires_grad=True)
        inv_freq, axis = P.rotary_frequencies((2,), device=DEV)
        for shape, ch in (((0, 4), -1), ((3, 0, 4), -1), ((0, 4, 5, 5), 1), ((2, 4, 0, 5), 1)):
            x = torch.empty(shape, dtype=dtype, device=DEV, requires_grad=True)
            for y, leaves in ((P.linear(x, w, b, activation="silu", channel_dim=ch), (x, w, b)),
                              (P.gated_linear(x, w, b, channel_dim=ch), (x, w, b)),
                              (P.layer_norm(x, n, n, channel_dim=ch), (x, n))):
                assert y.numel() == 0
                for leaf, g in zip(leaves, torch.autograd.grad(y, leaves, torch.zeros_like(y))):
                    assert g.shape == leaf.shape and not g.any()
        x = torch.empty(2, 0, 3, 4, dtype=dtype, device=DEV)
        assert P.rotary(x, inv_freq, axis, torch.empty(2, 0, 1, device=DEV)).shape == x.shape


def test_partial_gradients():
    """Only what is asked for is computed, and it is what the full backward gives."""
    import pwcnet_amd as P
    gen = _gen("partial")
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b = (_rand(gen, 50, 24, dtype=dtype), _rand(gen, 32, 24, dtype=dtype),
                   _rand(gen, 32, dtype=dtype))
        n = _rand(gen, 24, dtype=dtype)
        calls = [(lambda x, w, b: P.gated_linear(x, w, b, channel_dim=-1), (x, w, b), 16),
                 (lambda x, w, b: P.linear(x, w, b, activation="tanh", channel_dim=-1),
                  (x, w, b), 32),
                 (lambda x, w, b: P.linear(x, w, b, channel_dim=-1), (x, w, b), 32),
                 (lambda x, w, b: P.layer_norm(x, w, b, channel_dim=-1), (x, n, n.clone()), 24)]
        for call, leaves, out in calls:
            g = _rand(gen, 50, out, dtype=dtype)
            every = [t.clone().requires_grad_(True) for t in leaves]
            full = torch.autograd.grad(call(*every), every, g)
            for k in range(3):
                some = [t.clone().requires_grad_(i == k) for i, t in enumerate(leaves)]
                one, = torch.autograd.grad(call(*some), some[k], g)
                assert torch.equal(one, full[k])


def test_same_results_every_time():
    import pwcnet_amd as P
    gen = _gen("again")
    x = _rand(gen, 4, 96, 24, 28, dtype=torch.bfloat16).requires_grad_(True)
    blk = P.FeatureBlock(96).to(DEV, torch.bfloat16)
    g = _rand(gen, 4, 96, 24, 28, dtype=torch.bfloat16)
    first = None
    for _ in range(5):
        y = blk(x)
        got = [y.detach(), *torch.autograd.grad(y, [x, *blk.parameters()], g)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_other_stream_and_captured():
    """A forward and backward pass on a side stream, then captured: every replay, between eager
    passes and on new inputs, gives the eager results; two graphs do not share workspaces."""
    import pwcnet_amd as P
    gen = _gen("stream")
    blk = P.FeatureBlock(32).to(DEV)
    rot = P.RotaryPosition((0, 8, 8)).to(DEV)
    params = list(blk.parameters())
    shapes = [(2, 32, 12, 14), (3, 32, 9, 7)]

    def step(x, g):
        y = rot(blk(x), origin=(1, 0, 0))
        return [y.detach(), *torch.autograd.grad(y, [x, *params], g)]

    data = [[(_rand(gen, *s), _rand(gen, *s)) for _ in range(3)] for s in shapes]
    eager = [[step(x.clone().requires_grad_(True), g) for x, g in d] for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d, e in zip(data, eager):
            for (x, g), want in zip(d, e):
                got = step(x.clone().requires_grad_(True), g)
                side.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for s in shapes:
        xs, gs = torch.zeros(s, device=DEV, requires_grad=True), torch.zeros(s, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(xs, gs)
        graphs.append((graph, xs, gs, out))
    for turn in range(3):
        for (graph, xs, gs, out), d in zip(graphs, data):
            with torch.no_grad():
                xs.copy_(d[turn][0])
                gs.copy_(d[turn][1])
        graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for (graph, xs, gs, out), e in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(out, e[turn])), turn
        step(data[0][0][0].clone().requires_grad_(True), data[0][0][1])


def test_every_path_captured():
    """Products in parts, of few tokens, with rows laid out first and with two-part gradients, and
    norms of long rows: captured, and replayed on new inputs between eager calls."""
    import pwcnet_amd as P
    bf, hf = torch.bfloat16, torch.float16
    cases = [("gelu", False, (100, 2048), 520, bf), ("silu", True, (7, 1024), 200, bf),
             ("tanh", False, (301, 511), 509, bf), ("gelu", False, (3001, 517), 1021, bf),
             ("none", False, (64, 4096), 1200, hf), ("silu", True, (2, 96, 37, 53), 385, hf),
             ("norm", None, (301, 9216), 0, bf), ("norm", None, (2, 270, 21, 19), 0, hf)]

    def step(kind, gated, leaves, g):
        dim = -1 if leaves[0].dim() == 2 else 1
        if kind == "norm":
            y = P.layer_norm(*leaves, channel_dim=dim)
        elif gated:
            y = P.gated_linear(*leaves, activation=kind, channel_dim=dim)
        else:
            y = P.linear(*leaves, activation=kind, channel_dim=dim)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    for kind, gated, dims, O, dtype in cases:
        if kind == "norm":
            gen = _gen("captured", dims)
            C = dims[-1] if len(dims) == 2 else dims[1]
            made = [(_rand(gen, *dims, dtype=dtype), _rand(gen, C, dtype=dtype),
                     _rand(gen, C, dtype=dtype), _rand(gen, *dims, dtype=dtype)) for _ in range(2)]
        else:
            made = []
            for n in range(2):
                is_map = len(dims) == 4
                lead = (dims[0], *dims[2:]) if is_map else dims[:1]
                x, w, b, _, g = _product_case(is_map, lead, dims[1], O, dtype, kind, True, False,
                                              gated, seed=n)
                made.append((x, w, b, g))
        want = [step(kind, gated, [t.clone().requires_grad_(True) for t in m[:3]], m[3])
                for m in made]
        held = [t.clone().requires_grad_(True) for t in made[0][:3]]
        grad = made[0][3].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(kind, gated, held, grad)
        for turn in (1, 0, 1, 1):
            with torch.no_grad():
                for to, t in zip((*held, grad), made[turn]):
                    to.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[turn])), (kind, dims, turn)
            again = step(kind, gated, [t.clone().requires_grad_(True) for t in made[0][:3]],
                         made[0][3])
            assert all(torch.equal(a, b) for a, b in zip(again, want[0])), (kind, dims, turn)


def test_block_against_formula():
    """norm, gated, project with the skip, rotary: a run of them against 64 bits, with gradients.

    Bound by norms: each of the four outputs is rounded once (u, or fp32's sums), so a relative
    2-norm error of 8 u for 16 bits covers the chain forward and backward; fp32 2e-6."""
    import pwcnet_amd as P
    for dtype in DTYPES:
        gen = _gen("block", str(dtype))
        blk = P.FeatureBlock(64, 96).to(DEV, dtype)
        rot = P.RotaryPosition((0, 16, 16)).to(DEV)
        with torch.no_grad():
            for p in blk.parameters():
                p.add_(_rand(gen, *p.shape, dtype=dtype, scale=0.1))
        x = _rand(gen, 2, 64, 11, 13, dtype=dtype).requires_grad_(True)
        g = _rand(gen, 2, 64, 11, 13, dtype=dtype)
        y = rot(blk(x))
        grads = torch.autograd.grad(y, [x, *blk.parameters()], g)
        xd = x.detach().double().requires_grad_(True)
        ps = [p.detach().double().requires_grad_(True) for p in blk.parameters()]
        names = [n for n, _ in blk.named_parameters()]
        q = dict(zip(names, ps))
        t = _tok(xd, True)
        d = t - t.mean(1, keepdim=True)
        h = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * q["norm.weight"] + q["norm.bias"]
        z = h @ q["gated.weight"].t() + q["gated.bias"]
        h = z[:, :96] * torch.sigmoid(z[:, :96]) * z[:, 96:]
        t = t + h @ q["project.weight"].t() + q["project.bias"]
        n = torch.arange(11 * 13, device=DEV)
        at = torch.stack((0 * n, n // 13, n % 13), -1)
        a = at.double()[:, rot.axis.long()] * rot.inv_freq
        t = t.view(2, 143, 64)
        c, s = torch.cos(a), torch.sin(a)
        t = torch.cat((t[..., :32] * c - t[..., 32:] * s, t[..., :32] * s + t[..., 32:] * c), -1)
        ref = t.movedim(1, 2).reshape(2, 64, 11, 13)
        want = torch.autograd.grad(ref, [xd, *ps], g.double())
        tol = 2e-6 if dtype == torch.float32 else 8 * u(dtype)
        for name, a, b in zip(["y", "x", *names], [y, *grads], [ref, *want]):
            rel = ((a.double() - b).norm() / b.norm()).item()
            assert rel < tol, (dtype, name, rel)


def test_compiled_node_matches_eager():
    """The torch.ops.pwcnet nodes that tracers see give the eager values and gradients."""
    import pwcnet_amd as P  # noqa: F401  (registers the nodes)
    gen = _gen("nodes")
    x = _rand(gen, 2, 16, 5, 6).requires_grad_(True)
    w, b, g = _rand(gen, 16, 16), _rand(gen, 16), _rand(gen, 2, 16, 5, 6)
    n = _rand(gen, 16)
    g2 = g[:, :8].contiguous()
    inv_freq, axis = P.rotary_frequencies((4,), device=DEV)
    ops = torch.ops.pwcnet
    v = _rand(gen, 2, 6, 2, 8).requires_grad_(True)
    gv = _rand(gen, 2, 6, 2, 8)
    pairs = [(ops.linear(x, w, b, None, "gelu", 0.1, 1), P.linear(x, w, b, activation="gelu"), g, x),
             (ops.gated_linear(x, w, b, "silu", 0.1, 1), P.gated_linear(x, w, b), g2, x),
             (ops.layer_norm(x, n, b, 1e-5, 1)[0], P.layer_norm(x, n, b), g, x),
             (ops.rotary(v, inv_freq, axis, None, [2, 3], None, False, False),
              P.rotary(v, inv_freq, axis[:4], grid=(2, 3)), gv, v)]
    for a, c, grad, leaf in pairs:
        assert torch.equal(a, c)
        assert torch.equal(torch.autograd.grad(a, leaf, grad)[0],
                           torch.autograd.grad(c, leaf, grad)[0])


def test_net_with_refined_features():
    """Net's refined pyramid against the formula in 64 bits (2e-6 by norms, as the block above), and
    a forward and backward pass through all of it."""
    from pwcnet_amd.net import Net, NetArgs
    torch.manual_seed(3)
    args = NetArgs(feature_blocks=2, feature_rotary=True)
    net = Net(args).to(DEV)
    gen = _gen("net")
    pyr = [_rand(gen, 2, c, 2 << i, 3 << i) for i, c in enumerate(args.lv_chs[::-1])]
    with torch.no_grad():
        got = net.refine(pyr, 1)
    assert len(got) == 6 and got[5] is pyr[5]  # beyond the output level
    for l, (x, y) in enumerate(zip(pyr[:5], got)):
        t = _tok(x.double(), True)
        for blk in net.feature_refiners[l]:
            q = {n: p.detach().double() for n, p in blk.named_parameters()}
            d = t - t.mean(1, keepdim=True)
            h = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * q["norm.weight"]
            z = (h + q["norm.bias"]) @ q["gated.weight"].t() + q["gated.bias"]
            n = z.shape[1] // 2
            h = z[:, :n] * torch.sigmoid(z[:, :n]) * z[:, n:]
            t = t + h @ q["project.weight"].t() + q["project.bias"]
        rot = net.feature_rotaries[l]
        H, W = x.shape[2:]
        n = torch.arange(H * W, device=DEV)
        at = torch.stack((torch.ones_like(n), n // W, n % W), -1)[None]
        ref, _ = _rotary64(t.view(2, H * W, 1, -1), rot.inv_freq, rot.axis, at, False)
        ref = ref[:, :, 0].movedim(1, 2).reshape(x.shape)
        assert ((y.double() - ref).norm() / ref.norm()).item() < 2e-6
    # 128 x 128 is the least: at 64 x 64 the coarsest level is one pixel, where the warp's
    # flow / ((W - 1) / 2) is 0 / 0 whatever the features are
    x = torch.rand(1, 3, 2, 128, 128, generator=gen).to(DEV)
    flows, _ = net(x)
    sum(f.square().mean() for f in flows).backward()
    for name, p in net.named_parameters():
        if name.startswith("FeatureBlocks"):
            assert torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name


def test_refusals_on_the_device():
    """Shapes, types and places that the Python functions refuse, and a second derivative."""
    import pwcnet_amd as P
    x, w, b = (torch.zeros(2, 4, 3, 3, device=DEV), torch.zeros(6, 4, device=DEV),
               torch.zeros(6, device=DEV))
    f, a = P.rotary_frequencies((2,), device=DEV)
    h = torch.zeros(1, 9, 2, 4, device=DEV)
    for call, error, text in (
            (lambda: P.linear(x, w[:, :3]), ValueError, "weight shape"),
            (lambda: P.linear(x, w[0]), ValueError, "weight shape"),
            (lambda: P.linear(x, w[:0]), ValueError, "weight shape"),
            (lambda: P.linear(x, w, b[:5]), ValueError, "bias shape"),
            (lambda: P.linear(x, w, b, x), ValueError, "residual shape"),
            (lambda: P.linear(x, w, activation="swish"), ValueError, "activation"),
            (lambda: P.linear(x, w.half()), TypeError, "mixed dtypes"),
            (lambda: P.linear(x.double(), w.double()), TypeError, "unsupported dtype"),
            (lambda: P.linear(x, w.cpu()), RuntimeError, "HIP devices"),
            (lambda: P.linear(x, w, channel_dim=2), ValueError, "channel_dim"),
            (lambda: P.gated_linear(x, w[:5]), ValueError, "odd number"),
            (lambda: P.layer_norm(x, b), ValueError, "weight shape"),
            (lambda: P.layer_norm(x, eps=-1.0), ValueError, "eps"),
            (lambda: P.layer_norm(x[:, :0]), ValueError, "no channels"),
            (lambda: P.rotary(x[0], f, a, grid=(3,)), ValueError, "expected"),
            (lambda: P.rotary(h, f.float(), a, grid=(9,)), TypeError, "fp64"),
            (lambda: P.rotary(h, f, a.long(), grid=(9,)), TypeError, "int32"),
            (lambda: P.rotary(h[..., :3], f, a, grid=(9,)), ValueError, "pairs"),
            (lambda: P.rotary(h, f, a), ValueError, "positions or grid"),
            (lambda: P.rotary(h, f, a, f, grid=(9,)), ValueError, "positions or grid"),
            (lambda: P.rotary(h, f, a, grid=(2, 4)), ValueError, "grid"),
            (lambda: P.rotary(h, f, a, grid=(9,), origin=(1, 2)), ValueError, "grid"),
            (lambda: P.rotary(h, f, a, grid=(-3, -3)), ValueError, "grid"),
            (lambda: P.rotary(h, f, a, torch.zeros(8, 1, device=DEV)), ValueError, "positions"),
            (lambda: P.rotary(h, f, a, torch.zeros(9, 5, device=DEV)), ValueError, "positions"),
            (lambda: P.rotary(h, f, a, torch.zeros(9, 1, device=DEV).double()), TypeError,
             "positions"),
            (lambda: P.rotary(h, f, a, torch.zeros(9, 1)), RuntimeError, "different devices")):
        with pytest.raises(error, match=text):
            call()
    v = torch.randn(5, 4, device=DEV, requires_grad=True)
    for y in (P.linear(v, w, activation="silu", channel_dim=-1), P.gated_linear(v, w, channel_dim=-1),
              P.layer_norm(v, channel_dim=-1)):
        g, = torch.autograd.grad(y.square().sum(), v, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiat"):
            g.sum().backward()


def test_threads_and_inplace_changes():
    """Two threads at once, and a saved input that was changed before its backward pass."""
    import threading
    import pwcnet_amd as P
    gen = _gen("threads")
    x, w, g = _rand(gen, 64, 48), _rand(gen, 32, 48), _rand(gen, 64, 32)

    def step(stream):
        with torch.cuda.stream(stream):
            a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            y = P.linear(a, b, activation="gelu", channel_dim=-1)
            out = [y.detach(), *torch.autograd.grad(y, (a, b), g)]
            stream.synchronize()
            return out

    want = step(torch.cuda.current_stream())
    got = {}

    def work(k):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        for _ in range(20):
            got[k] = step(s)
            assert all(torch.equal(p, q) for p, q in zip(got[k], want))
        got[k] = "done"

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got == {0: "done", 1: "done"}
    a = x.clone().requires_grad_(True)
    c = a * 1
    y = P.linear(c, w, activation="gelu", channel_dim=-1)
    with torch.no_grad():
        c.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_images_of_one_pixel_are_tokens():
    """[B, C, 1, 1] gives the values and gradients of [B, C], from a strided batch too."""
    import pwcnet_amd as P
    for dtype in DTYPES:
        gen = _gen("pixel", str(dtype))
        w, b, g = (_rand(gen, 96, 40, dtype=dtype, scale=0.2), _rand(gen, 96, dtype=dtype),
                   _rand(gen, 70, 48, dtype=dtype))
        wide = _rand(gen, 70, 43, dtype=dtype)
        for x in (wide[:, :40].contiguous(), wide[:, 3:]):
            got = []
            for shape, dim in (((70, 40), -1), ((70, 40, 1, 1), 1)):
                v = x.detach().reshape(70, 40) if dim == -1 else x.detach()[:, :, None, None]
                leaves = [v.requires_grad_(True), w.clone().requires_grad_(True),
                          b.clone().requires_grad_(True)]
                n = P.layer_norm(leaves[0], channel_dim=dim)
                y = P.gated_linear(n, *leaves[1:], channel_dim=dim)
                assert y.shape == (70, 48, *shape[2:])
                grads = torch.autograd.grad(y, leaves, g.reshape(y.shape))
                got.append([t.reshape(70, -1) if t.shape[0] == 70 else t for t in (y, *grads)])
            assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(*got))


def test_offsets_past_32_bits():
    """More than 2^31 values: the last rows equal a call on them alone."""
    import pwcnet_amd as P
    M, C, last = 2 ** 20 + 70, 2056, 66
    x = torch.empty(M, C, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(5))
    gen = _gen("far")
    w = _rand(gen, 24, C, dtype=torch.bfloat16, scale=C ** -0.5)
    b = _rand(gen, C, dtype=torch.bfloat16)
    assert torch.equal(P.layer_norm(x, b, b, channel_dim=-1)[-last:],
                       P.layer_norm(x[-last:], b, b, channel_dim=-1))
    inv, axis = P.rotary_frequencies((C // 8,), device=DEV)
    at = torch.arange(M, device=DEV)[:, None]
    assert torch.equal(P.rotary(x.view(1, M, 4, C // 4), inv, axis, at)[:, -last:],
                       P.rotary(x[-last:].view(1, last, 4, C // 4), inv, axis, at[-last:]))
    # (the whole and the part may take other kernels: sums of the same products in another order)
    whole, part = P.linear(x, w, channel_dim=-1)[-last:], P.linear(x[-last:], w, channel_dim=-1)
    bound = x[-last:].float().abs() @ w.float().abs().t()
    _within("linear", whole, part, 2 * C * F32 * bound
            + 2 * u(torch.bfloat16) * (part.abs().float() + 2 * C * F32 * bound))
    dy = _rand(gen, M, 24, dtype=torch.bfloat16)
    from pwcnet_amd import features
    gx = features.linear_backward(x, w, None, dy, channel_dim=-1, needs=(True, False, False))[0]
    ref = dy[-last:].double() @ w.double()
    tol = 26 * F32 * (dy[-last:].double().abs() @ w.double().abs())
    _within("dx", gx[-last:], ref, tol + u(torch.bfloat16) * (ref.abs() + tol))
    del gx, whole
    # a map whose image is that large
    m, v = x.view(-1)[: 2 ** 31 + 64].view(1, 2, -1), _rand(gen, 3, 2, dtype=torch.bfloat16)
    assert torch.equal(P.linear(m, v)[..., -64:], P.linear(m[..., -64:].contiguous(), v))
    assert torch.equal(P.layer_norm(m)[..., -64:], P.layer_norm(m[..., -64:].contiguous()))


def test_derivatives_that_there_are_not():
    """Forward-mode derivatives and negated views are refused, not dropped."""
    import torch.autograd.forward_ad as fwad
    import pwcnet_amd as P
    x, w = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV)
    inv, axis = P.rotary_frequencies((4,), device=DEV)
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: P.layer_norm(d, channel_dim=-1), lambda: P.linear(d, w, channel_dim=-1),
                     lambda: P.gated_linear(x, fwad.make_dual(w, w), channel_dim=-1),
                     lambda: P.rotary(d[None, :, None], inv, axis, grid=(4,))):
            with pytest.raises(RuntimeError):
                call()
    neg = torch.conj(torch.randn(1, 4, 1, 8, dtype=torch.complex64, device=DEV)).imag
    with pytest.raises(TypeError, match="negated"):
        P.rotary(neg, inv, axis, grid=(4,))
    assert torch.equal(P.rotary(neg.resolve_neg(), inv, axis, grid=(4,)),
                       P.rotary(neg.clone(), inv, axis, grid=(4,)))


def test_dispatch_modes_see_single_nodes():
    """Under a dispatch mode an eager call shows as its node."""
    from torch.utils._python_dispatch import TorchDispatchMode
    import pwcnet_amd as P

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    seen = []
    x, w = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV)
    want = P.linear(x, w, activation="gelu", channel_dim=-1)
    with Names():
        got = P.linear(x, w, activation="gelu", channel_dim=-1)
    assert torch.equal(got, want) and any("pwcnet.linear" in n for n in seen)


def test_rotary_entry_turns_in_place():
    """y == x with equal strides; a second call with `inverse` turns back."""
    import ctypes
    import pwcnet_amd as P
    from pwcnet_amd import _lib
    lib = _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        for shape, perm, pairs in (((2, 9, 6, 64), (0, 1, 2, 3), 24),
                                   ((2, 6, 20, 35), (0, 3, 1, 2), 10)):
            base = _rand(_gen("in place", str(dtype), shape), *shape, dtype=dtype)
            x = base.permute(*perm)
            inv, axis = P.rotary_frequencies((pairs,), device=DEV)
            want = P.rotary(x, inv, axis, grid=(x.shape[1],))
            s = _lib.RotaryShape(B=x.shape[0], N=x.shape[1], heads=x.shape[2], D=x.shape[3],
                                 pairs=pairs, axes=1)
            s.x_stride[:] = s.y_stride[:] = x.stride()
            s.grid[:] = [x.shape[1], 0, 0, 0]
            _lib.check(lib.pwc_rotary(x.data_ptr(), x.data_ptr(), None, inv.data_ptr(),
                                      axis.data_ptr(), ctypes.byref(s), 0, code, stream), "rotary")
            assert torch.equal(x, want)
            back = P.features.rotary_forward(want, inv, axis, grid=(x.shape[1],), inverse=True)
            _lib.check(lib.pwc_rotary(x.data_ptr(), x.data_ptr(), None, inv.data_ptr(),
                                      axis.data_ptr(), ctypes.byref(s), 1, code, stream), "rotary")
            assert torch.equal(x, back)


@pytest.mark.parametrize("layout,B,P_,K,O,gated,act", [
    (1, 1, 100, 2048, 520, 0, 6), (1, 1, 7, 1024, 131, 1, 5), (1, 1, 301, 511, 509, 0, 4),
    (1, 1, 3001, 517, 1021, 1, 5), (0, 2, 1961, 96, 385, 1, 6), (0, 3, 35, 33, 17, 0, 0),
    (1, 1, 64, 4096, 1200, 0, 0), (0, 5, 1, 40, 24, 1, 5)])
def test_entries_stay_in_their_buffers(layout, B, P_, K, O, gated, act):
    """Outputs and a workspace of exactly the asked size stand between values that stay as they were;
    each subset of the gradients gives the full call's."""
    import ctypes
    from pwcnet_amd import _lib
    lib = _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    gen = _gen("buffers", layout, B, P_, K, O, gated)
    rows, M = O * (2 if gated else 1), B * P_
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        x, w = (_rand(gen, M, K, dtype=dtype), _rand(gen, rows, K, dtype=dtype, scale=K ** -0.5))
        b, dy = _rand(gen, rows, dtype=dtype), _rand(gen, M, O, dtype=dtype)
        stride = K if layout == 1 else K * P_
        guard = 4096

        def buffer(values, size):
            buf = torch.full((values * size + 2 * guard,), 0x5A, dtype=torch.uint8, device=DEV)
            return buf, buf.data_ptr() + guard

        def kept(buf, used):
            return bool((buf[:guard] == 0x5A).all()) and bool((buf[guard + used:] == 0x5A).all())

        size = dtype.itemsize
        name = "gated_linear" if gated else "linear"
        asked = getattr(lib, f"pwc_{name}_forward_workspace_size")(
            x.data_ptr(), w.data_ptr(), layout, B, P_, K, O, stride, code)
        y, at = buffer(M * O, size)
        ws, ws_at = buffer(asked, 1)
        middle = () if gated else (None,)
        _lib.check(getattr(lib, f"pwc_{name}_forward")(
            x.data_ptr(), w.data_ptr(), b.data_ptr(), *middle, at, layout, B, P_, K, O, stride, act,
            0.1, code, ws_at, asked, stream), name)
        torch.cuda.synchronize()
        assert kept(y, M * O * size) and kept(ws, asked)
        back_size = getattr(lib, f"pwc_{name}_backward_workspace_size")
        asked = back_size(x.data_ptr(), w.data_ptr(), dy.data_ptr(), layout, B, P_, K, O, stride,
                          *(() if gated else (act,)), code)
        full = None
        for which in (7, 1, 2, 4, 3, 5, 6):
            outs = [buffer(n, size) for n in (M * K, rows * K, rows)]
            ws, ws_at = buffer(asked, 1)
            _lib.check(getattr(lib, f"pwc_{name}_backward")(
                x.data_ptr(), w.data_ptr(), b.data_ptr(), dy.data_ptr(),
                *(o[1] if which >> k & 1 else None for k, o in enumerate(outs)), layout, B, P_, K, O,
                stride, act, 0.1, code, ws_at, asked, stream), name)
            torch.cuda.synchronize()
            assert kept(ws, asked)
            for o, n in zip(outs, (M * K, rows * K, rows)):
                assert kept(o[0], n * size)
            full = full or [o[0].clone() for o in outs]
            for k, o in enumerate(outs):
                if which >> k & 1:
                    assert torch.equal(o[0], full[k]), (which, k)
                else:
                    assert bool((o[0] == 0x5A).all())
