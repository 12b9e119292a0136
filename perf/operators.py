"""Cases of the feature operators: layer norm, rotary positions, linear and gated linear.

Each case is one call of an operator as a program around the correlation makes it: on feature maps
[B, C, H, W] (``layout`` "map") or on tokens [N, C] ("tokens"), forward alone or with its backward
pass (``train``).  With ``own`` false ``run`` computes the operator from elementary torch operations
in 32 bits (angles in 64), rounded once at the end; with ``own`` true it calls pwcnet_amd.
"""
import math
import os
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_SMOOTH = ("none", "silu", "gelu", "gelu_tanh", "sigmoid", "tanh")
_KINKED = ("relu", "leaky_relu")


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token of a decoder: nothing but latency
        dict(name="norm_one", op="norm", layout="tokens", dtype="bf16", tokens=1, channels=1024,
             train=False),
        # the l4 feature map of the 384x448 training step
        dict(name="norm_map_l4", op="norm", layout="map", dtype="fp32", batch=8, height=96,
             width=112, channels=32, train=True),
        # a training batch of tokens, one short of a round count
        dict(name="norm_tokens", op="norm", layout="tokens", dtype="bf16", tokens=16383,
             channels=2048, train=True),
        # four sequences' next token, far into a video
        dict(name="rotary_one", op="rotary", layout="tokens", dtype="bf16", batch=4, tokens=1,
             heads=32, channels=128, rotated=64, axes=3, interleaved=False, train=False),
        # the l4 map of 448x1024 frames, positions from its grid
        dict(name="rotary_map_l4", op="rotary", layout="map", dtype="fp16", batch=16, height=112,
             width=256, heads=1, channels=32, rotated=16, axes=2, interleaved=False, train=False),
        # the queries of two clips of patches, with positions in hand
        dict(name="rotary_video", op="rotary", layout="tokens", dtype="bf16", batch=2,
             tokens=9603, heads=24, channels=128, rotated=64, axes=3, interleaved=True,
             train=True),
        # one new token through a square projection: the weights are read once
        dict(name="linear_one", op="linear", layout="tokens", dtype="bf16", tokens=1,
             channels=4096, out=4096, act="none", bias=True, residual=True, train=False),
        # a 1x1 convolution with LeakyReLU and skip on the l3 map
        dict(name="linear_map_l3", op="linear", layout="map", dtype="fp32", batch=8, height=48,
             width=56, channels=64, out=64, act="leaky_relu", bias=True, residual=True,
             train=False),
        # a training batch through a widening projection
        dict(name="linear_tokens", op="linear", layout="tokens", dtype="bf16", tokens=8192,
             channels=1024, out=4096, act="gelu", bias=True, residual=False, train=True),
        # seven tokens of a decoder's batch
        dict(name="gated_few", op="gated", layout="tokens", dtype="bf16", tokens=7,
             channels=2048, out=5632, act="silu", bias=False, train=False),
        # a block on odd-sized maps of l2's channels
        dict(name="gated_map_odd", op="gated", layout="map", dtype="fp16", batch=5, height=37,
             width=53, channels=96, out=385, act="gelu_tanh", bias=True, train=True),
        # a training batch through the block
        dict(name="gated_tokens", op="gated", layout="tokens", dtype="bf16", tokens=8192,
             channels=1024, out=4096, act="silu", bias=True, train=True),
    ]


def _spread(rng, lo, hi):
    """A whole number, uniform in its logarithm; half of them rounded to a multiple of 8."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    v = min(hi, max(lo, int(v)))
    return max(lo, v // 8 * 8) if rng.random() < 0.5 and v >= 8 else v


def draw(rng):
    most = max((work(c)["bytes"], work(c)["flops"]) for c in listed())
    flops = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(("norm", "rotary", "linear", "gated"))
        c = dict(op=op, layout=rng.choice(("map", "tokens")),
                 dtype=rng.choice(("fp32", "fp16", "bf16")), train=rng.random() < 0.5)
        if c["layout"] == "map":
            c.update(batch=rng.randint(1, 16), height=_spread(rng, 1, 112),
                     width=_spread(rng, 1, 256))
        else:
            c.update(tokens=_spread(rng, 1, 16384))
        if op == "rotary":
            c["channels"] = 2 * _spread(rng, 2, 64)
            half = c["channels"] // 2
            c.update(heads=_spread(rng, 1, 32), axes=rng.randint(1, 3),
                     rotated=half if rng.random() < 0.7 else rng.randint(1, half),
                     interleaved=rng.random() < 0.5)
            c.setdefault("batch", rng.randint(1, 4))
        else:
            c["channels"] = _spread(rng, 1, 256 if c["layout"] == "map" else 4096)
        if op in ("linear", "gated"):
            c["out"] = _spread(rng, 1, 1024 if c["layout"] == "map" else 8192)
            # two right programs may differ by a whole step of the derivative where z is within
            # their rounding of a kink: that shows in 32 bits, so those gradients are smooth ones
            c["act"] = rng.choice(_SMOOTH if c["train"] and c["dtype"] == "fp32"
                                  else _SMOOTH + _KINKED)
            c["bias"] = rng.random() < 0.7
        if op == "linear":
            c["residual"] = rng.random() < 0.5
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= flops:
            return c


# ------------------------------------------------------------------------------- their work
def _tokens(c):
    if c["layout"] == "map":
        return c["batch"] * c["height"] * c["width"]
    return c["tokens"] * (c["batch"] if c["op"] == "rotary" else 1)


def work(c):
    m, k, s = _tokens(c), c["channels"], _SIZE[c["dtype"]]
    if c["op"] == "norm":
        n = m * k
        return {"bytes": s * (5 * n + 4 * k if c["train"] else 2 * n + 2 * k),
                "flops": (18 if c["train"] else 8) * n}
    if c["op"] == "rotary":
        n = m * k * c["heads"]
        passes = 2 if c["train"] else 1
        at = 0 if c["layout"] == "map" else 8 * m * c["axes"]
        return {"bytes": passes * (2 * n * s + at), "flops": passes * 3 * n}
    o = c["out"]
    rows = 2 * o if c["op"] == "gated" else o
    values = m * k + m * o + rows * k + (rows if c["bias"] else 0)
    values += m * o if c.get("residual") else 0
    if c["train"]:  # the output's gradient in, the gradients of x, weight and bias out
        values += m * o + m * k + rows * k + (rows if c["bias"] else 0)
    return {"bytes": s * values, "flops": 2 * m * k * rows * (3 if c["train"] else 1)}


# ------------------------------------------------------------------------------- the inputs
def _inv_freq(c):
    """Each axis gets its own ladder of frequencies 10000^(-j / n), n of the rotated pairs."""
    r, a = c["rotated"], c["axes"]
    axis = torch.arange(r, device="cuda") * a // r
    first = (axis[:, None] == torch.arange(a, device="cuda")).sum(0)
    start = torch.cumsum(first, 0) - first
    j = torch.arange(r, device="cuda") - start[axis]
    return 10000.0 ** (-j.double() / first[axis].double()), axis.to(torch.int32)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def feature(*shape):  # what a LeakyReLU(0.1) lets through, off centre
        v = randn(*shape)
        return torch.where(v > 0, v, 0.1 * v).to(dt)

    s = dict(c)
    lead = (c["batch"], c["height"], c["width"]) if c["layout"] == "map" else (c["tokens"],)

    def shaped(n, make):
        if c["layout"] == "map":
            return make(lead[0], n, lead[1], lead[2])
        return make(lead[0], n)

    k = c["channels"]
    if c["op"] == "rotary":
        s["inv_freq"], s["axis"] = _inv_freq(c)
        if c["layout"] == "map":
            s["x"] = feature(c["batch"], c["heads"] * k, c["height"], c["width"])
        else:
            s["x"] = randn(c["batch"], c["tokens"], c["heads"], k).to(dt)
            s["positions"] = torch.randint(0, 4096, (c["batch"], c["tokens"], c["axes"]),
                                           generator=gen, device="cuda")
        if c["train"]:
            s["g"] = randn(*s["x"].shape).to(dt)
    else:
        s["x"] = shaped(k, feature)
        if c["op"] == "norm":
            s["w"] = (1 + 0.1 * randn(k)).to(dt)
            s["b"] = (0.1 * randn(k)).to(dt)
            o = k
        else:
            o = c["out"]
            rows = 2 * o if c["op"] == "gated" else o
            s["w"] = (randn(rows, k) / math.sqrt(k)).to(dt)
            s["b"] = (0.1 * randn(rows)).to(dt) if c["bias"] else None
            s["res"] = shaped(o, feature) if c.get("residual") else None
        if c["train"]:
            s["g"] = shaped(o, randn).to(dt)
    if c["train"]:
        for name in ("x", "w", "b", "res"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------- the plain forms
def _act(z, name, slope=0.1):
    """(act(z), act'(z))"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if name == "leaky_relu":
        d = torch.where(z > 0, torch.ones_like(z), torch.full_like(z, slope))
        return z * d, d
    if name == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return p, p * (1 - p)
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 0.134145 * z * z)


def _plain_norm(s, dt):
    ch = 1 if s["layout"] == "map" else -1
    along = (1, -1, 1, 1) if s["layout"] == "map" else (-1,)
    rest = (0, 2, 3) if s["layout"] == "map" else (0,)
    x, w, b = s["x"].float(), s["w"].float().view(along), s["b"].float().view(along)
    d = x - x.mean(ch, keepdim=True)
    r = 1 / torch.sqrt((d * d).mean(ch, keepdim=True) + 1e-5)
    xh = d * r
    out = {"y": (xh * w + b).to(dt)}
    if s["train"]:
        g = s["g"].float()
        gw = g * w
        dx = r * (gw - gw.mean(ch, keepdim=True) - xh * (gw * xh).mean(ch, keepdim=True))
        out.update(dx=dx.to(dt), dw=(g * xh).sum(rest).to(dt), db=g.sum(rest).to(dt))
    return out


def _plain_turn(s, x, sign, dt):
    """x: [B, N, heads, D]"""
    r = s["rotated"]
    if s["layout"] == "map":
        n = torch.arange(s["height"] * s["width"], device=x.device)
        yx = (torch.zeros_like(n), n // s["width"], n % s["width"])
        at = torch.stack(yx[-s["axes"]:] if s["axes"] > 1 else (n,), -1)[None]
    else:
        at = s["positions"]
    a = at.double()[..., s["axis"].long()] * s["inv_freq"]
    cos, sin = torch.cos(a).float()[:, :, None], (sign * torch.sin(a)).float()[:, :, None]
    x = x.float()
    y = x.clone()
    u = slice(0, 2 * r, 2) if s["interleaved"] else slice(0, r)
    v = slice(1, 2 * r, 2) if s["interleaved"] else slice(r, 2 * r)
    y[..., u] = x[..., u] * cos - x[..., v] * sin
    y[..., v] = x[..., u] * sin + x[..., v] * cos
    return y.to(dt)


def _heads_last(s, x):
    """A map [B, heads * D, H, W] as [B, N, heads, D]; tokens are that already."""
    if s["layout"] == "map":
        return x.reshape(s["batch"], s["heads"], s["channels"], -1).permute(0, 3, 1, 2)
    return x


def _heads_first(s, y):
    if s["layout"] == "map":
        return y.permute(0, 2, 3, 1).reshape(s["batch"], -1, s["height"], s["width"])
    return y


def _plain_rotary(s, dt):
    out = {"y": _heads_first(s, _plain_turn(s, _heads_last(s, s["x"]), 1, dt))}
    if s["train"]:
        out["dx"] = _heads_first(s, _plain_turn(s, _heads_last(s, s["g"]), -1, dt))
    return out


def _by_channel(s, v):
    """Tokens [N, C], or a map [B, C, H, W] as [B, C, H * W]."""
    return v.flatten(2) if s["layout"] == "map" else v


def _plain_products(s, dt):
    """linear and gated linear."""
    as_map = s["layout"] == "map"
    x, w = _by_channel(s, s["x"].float()), s["w"].float()
    z = torch.matmul(w, x) if as_map else torch.matmul(x, w.t())
    if s["b"] is not None:
        z = z + (s["b"].float()[:, None] if as_map else s["b"].float())
    ch = 1 if as_map else -1
    gated = s["op"] == "gated"
    if gated:
        zg, zu = z.chunk(2, ch)
        f, df = _act(zg, s["act"])
        y = f * zu
    else:
        f, df = _act(z, s["act"])
        y = f if s["res"] is None else f + _by_channel(s, s["res"].float())
    shape = list(s["x"].shape)
    shape[ch] = s["out"]
    out = {"y": y.to(dt).view(shape)}
    if s["train"]:
        g = _by_channel(s, s["g"].float())
        dz = torch.cat((g * zu * df, g * f), ch) if gated else g * df
        if as_map:
            out["dx"] = torch.matmul(w.t(), dz)
            out["dw"] = torch.matmul(dz, x.transpose(1, 2)).sum(0)
            out["db"] = dz.sum((0, 2))
        else:
            out["dx"] = torch.matmul(dz, w)
            out["dw"] = torch.matmul(dz.t(), x)
            out["db"] = dz.sum(0)
        out = {n: v.to(dt) for n, v in out.items()}
        out["dx"] = out["dx"].view(s["x"].shape)
        if s["b"] is None:
            del out["db"]
        if s.get("res") is not None:
            out["dres"] = s["g"]
    return out


# ------------------------------------------------------------------------------- the framework's
def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "pwc-net_pytorch_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import pwcnet_amd
    return pwcnet_amd


def _own(s):
    P = _framework()
    ch = 1 if s["layout"] == "map" else -1
    x = s["x"]
    if s["op"] == "norm":
        y = P.layer_norm(x, s["w"], s["b"], eps=1e-5, channel_dim=ch)
    elif s["op"] == "linear":
        y = P.linear(x, s["w"], s["b"], s["res"], activation=s["act"], negative_slope=0.1,
                     channel_dim=ch)
    elif s["op"] == "gated":
        y = P.gated_linear(x, s["w"], s["b"], activation=s["act"], negative_slope=0.1,
                           channel_dim=ch)
    elif s["layout"] == "map":
        h, w = s["height"], s["width"]
        grid = (h * w,) if s["axes"] == 1 else (h, w) if s["axes"] == 2 else (1, h, w)
        y = P.rotary(x.view(s["batch"], s["heads"], s["channels"], h * w).permute(0, 3, 1, 2),
                     s["inv_freq"], s["axis"], grid=grid, interleaved=s["interleaved"])
        y = y.permute(0, 2, 3, 1).reshape(x.shape)
    else:
        y = P.rotary(x, s["inv_freq"], s["axis"], s["positions"], interleaved=s["interleaved"])
    if not s["train"]:
        return {"y": y}
    names = [n for n in ("x", "w", "b", "res") if s.get(n) is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["g"])
    return {"y": y.detach(), **{"d" + n: v for n, v in zip(names, grads)}}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        dt = _DT[state["dtype"]]
        if state["op"] == "norm":
            return _plain_norm(state, dt)
        if state["op"] == "rotary":
            return _plain_rotary(state, dt)
        return _plain_products(state, dt)


# ------------------------------------------------------------------------------- in 64 bits
def _exact_phi(z, name):
    """The activation of a float64 tensor, differentiable."""
    zero = torch.zeros_like(z)
    if name == "relu":
        return torch.maximum(z, zero)
    if name == "leaky_relu":
        return torch.maximum(z, zero) + 0.1 * torch.minimum(z, zero)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":  # (1 + tanh a) / 2 = sigmoid(2 a)
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def exact(case, seed):
    s = prepare(case, seed)
    as_map = s["layout"] == "map"
    leaf = {n: s[n].detach().double().requires_grad_(True)
            for n in ("x", "w", "b", "res") if s.get(n) is not None}
    x = leaf["x"]
    if s["op"] == "rotary":
        # complex numbers times e^(i angle)
        b, heads, d, r = s["batch"], s["heads"], s["channels"], s["rotated"]
        if as_map:
            h, w = s["height"], s["width"]
            at = torch.cartesian_prod(torch.arange(h), torch.arange(w)).reshape(-1, 2).double()
            if s["axes"] == 1:
                at = torch.arange(h * w).double()[:, None]
            elif s["axes"] == 3:
                at = torch.cat((torch.zeros(h * w, 1, dtype=torch.float64), at), 1)
            at = at.cuda()[None]
            v = x.reshape(b, heads, d, h * w).movedim(3, 1)
        else:
            at, v = s["positions"].double(), x
        angle = torch.gather(at, 2, s["axis"].long().expand(*at.shape[:2], r)) * s["inv_freq"]
        if s["interleaved"]:
            pair = v[..., :2 * r].reshape(*v.shape[:3], r, 2)
        else:
            pair = v[..., :2 * r].reshape(*v.shape[:3], 2, r).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pair.contiguous())
                                    * torch.polar(torch.ones_like(angle), angle)[:, :, None])
        if not s["interleaved"]:
            turned = turned.transpose(-1, -2)
        y = torch.cat((turned.reshape(*v.shape[:3], 2 * r), v[..., 2 * r:]), -1)
        y = y.movedim(1, 3).reshape(x.shape) if as_map else y
    elif s["op"] == "norm":
        v = x.movedim(1, -1) if as_map else x
        var, mu = torch.var_mean(v, -1, correction=0, keepdim=True)
        y = (v - mu) * torch.rsqrt(var + 1e-5) * leaf["w"] + leaf["b"]
        y = y.movedim(-1, 1) if as_map else y
    else:
        v = x.movedim(1, -1).reshape(-1, x.shape[1]) if as_map else x
        z = torch.mm(v, leaf["w"].t())
        z = z + leaf["b"] if s["b"] is not None else z
        if s["op"] == "gated":
            y = _exact_phi(z[:, :s["out"]], s["act"]) * z[:, s["out"]:]
        else:
            y = _exact_phi(z, s["act"])
        if as_map:
            y = y.reshape(s["batch"], s["height"], s["width"], -1).movedim(-1, 1)
        y = y + leaf["res"] if s.get("res") is not None else y
    if not s["train"]:
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, list(leaf.values()), s["g"].double())
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(leaf, grads)}}
