"""Performance cases of the operators around the attention of a rope-DiT block: adaLN layer norm, projections with their epilogues, and
rotary positions over several axes.

A case is one pass through one operator: the forward alone (sampling) or the forward and the gradients of every input (training).  Keys:

    op      layer_norm | linear | rope_axes
    pass    fwd | train
    dtype   bf16 | fp32

    layer_norm  B, N, C   samples, tokens of each, channels;  affine: learned weight and bias;  modulated: a scale and a shift per sample
    linear      B, N, K, F  samples, tokens of each, input and output features;  act: none | gelu_tanh | silu;  bias;  residual: y = residual + (...);
                gate: a factor per sample and output feature in front of the residual
    rope_axes   B, H, N, D;  axes: channels of each axis;  positions: grid | far | fractional, per_sample: positions of each sample;
                layout: bhnd | bnhd ([B,H,N,D] views of [B,N,H,D] storage, what a projection hands over)

`own` False: the operators written out in torch.  `own` True: the calls that a program makes of this package.
"""
import math

import torch

own = False

EPS = 1e-6
THETA = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(mode, B, N, C, affine=False, modulated=True, dtype="bf16", name=None):
    c = {"op": "layer_norm", "pass": mode, "dtype": dtype, "B": B, "N": N, "C": C, "affine": affine, "modulated": modulated}
    return dict(c, name=name) if name else c


def _linear(mode, B, N, K, F, act="none", bias=True, residual=False, gate=False, dtype="bf16", name=None):
    c = {"op": "linear", "pass": mode, "dtype": dtype, "B": B, "N": N, "K": K, "F": F, "act": act, "bias": bias, "residual": residual, "gate": gate}
    return dict(c, name=name) if name else c


def _rope(mode, B, H, N, axes, positions="grid", per_sample=False, layout="bnhd", dtype="bf16", name=None):
    c = {"op": "rope_axes", "pass": mode, "dtype": dtype, "B": B, "H": H, "N": N, "D": sum(axes), "axes": ",".join(map(str, axes)),
         "positions": positions, "per_sample": per_sample, "layout": layout}
    return dict(c, name=name) if name else c


def listed():
    return [
        # adaLN in front of the attention: one denoising step of one image on a 32 x 32 latent, the smallest call of a sampling program
        _norm("fwd", 1, 1024, 384, name="norm 32x32 sample"),
        # the same in a training step at 128 x 128 tokens, eight images
        _norm("train", 8, 16384, 384, name="norm 128x128 train"),
        # a layer norm with learned weight and bias in fp32, rows of no whole number of vectors, a ragged length
        _norm("train", 3, 5377, 1155, affine=True, modulated=False, dtype="fp32", name="norm affine ragged fp32 train"),
        # a wider model: learned and modulated at once, a short sequence
        _norm("train", 2, 1001, 2048, affine=True, name="norm wide train"),
        # the first projection of the timestep embedding: one row per image
        _linear("fwd", 8, 1, 256, 384, act="silu", name="linear timestep sample"),
        # the feed-forward's first projection while sampling one image at 128 x 128 tokens
        _linear("fwd", 1, 16384, 384, 1536, act="gelu_tanh", name="linear ff in sample"),
        # the same in a training step of eight images
        _linear("train", 8, 16384, 384, 1536, act="gelu_tanh", name="linear ff in train"),
        # the feed-forward's second projection: gated, onto the residual stream
        _linear("train", 8, 16384, 1536, 384, residual=True, gate=True, name="linear ff out train"),
        # odd widths and a ragged length, onto a residual without a gate
        _linear("train", 3, 1001, 389, 771, residual=True, name="linear ragged train"),
        # the attention's output projection in fp32, as a numerics check runs it
        _linear("train", 2, 1024, 384, 384, residual=True, gate=True, dtype="fp32", name="linear out fp32 train"),
        # rows and columns of an image, eight images at 128 x 128 tokens
        _rope("train", 8, 6, 16384, (32, 32), name="rope 128x128 train"),
        # time, rows and columns of a clip in fp32, positions of each sample far from the origin (a window of a long video)
        _rope("fwd", 2, 3, 5001, (16, 24, 24), positions="far", per_sample=True, layout="bhnd", dtype="fp32", name="rope video fp32 sample"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6e12, w["flops"] / (5e13 if c["dtype"] == "fp32" else 1.4e15))


def _width(rng, lo, hi):
    """A feature count: half of them whole multiples of 64, the others anything."""
    n = _spread(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(("layer_norm", "linear", "linear", "rope_axes"))
        mode, dtype = rng.choice(("fwd", "train", "train")), "fp32" if rng.random() < 0.2 else "bf16"
        B, N = _spread(rng, 1, 16), _spread(rng, 1, 16384)
        if op == "layer_norm":
            c = _norm(mode, B, N, _width(rng, 8, 4096), rng.random() < 0.5, rng.random() < 0.6, dtype)
        elif op == "linear":
            residual = rng.random() < 0.5
            gate = residual and rng.random() < 0.6
            act = "none" if gate else rng.choice(("none", "gelu_tanh", "silu"))
            c = _linear(mode, B, N, _width(rng, 16, 2048), _width(rng, 16, 2048), act, rng.random() < 0.8, residual, gate, dtype)
        else:
            axes = rng.choice(((64,), (32, 32), (16, 24, 24), (64, 64), (32, 48, 48), (8, 12, 12), (16, 56, 56)))
            c = _rope(mode, B, _spread(rng, 1, 16), N, axes, rng.choice(("grid", "grid", "far", "fractional")), rng.random() < 0.3,
                      rng.choice(("bhnd", "bnhd")), dtype)
        if _cost(c) <= most[op]:
            return c


def _places(c, gen, dev):
    """Positions of the tokens on every axis: [N, A], or [B, N, A] where every sample has its own."""
    N, A = c["N"], len(_axes(c))
    side = max(1, math.ceil(N ** (1.0 / A) - 1e-9))
    n = torch.arange(N, device=dev)
    grid = torch.stack([torch.div(n, side ** (A - 1 - a), rounding_mode="floor") % side if a else torch.div(n, side ** (A - 1), rounding_mode="floor")
                        for a in range(A)], -1)
    lead = (c["B"], 1, 1) if c["per_sample"] else (1, 1)
    if c["positions"] == "far":          # a window that begins somewhere in a long sequence
        grid = grid + torch.randint(0, 1 << 20, lead[:-1] + (A,), generator=gen, device=dev)
    elif c["positions"] == "fractional":      # positions of another resolution, interpolated
        grid = grid * 0.37 + torch.rand(lead[:-1] + (A,), generator=gen, device=dev)
    elif c["per_sample"]:                # crops of one image
        grid = grid + torch.randint(0, 64, lead[:-1] + (A,), generator=gen, device=dev)
    return grid.float().contiguous() if c["positions"] == "fractional" else grid.contiguous()


def _axes(c):
    return tuple(int(a) for a in c["axes"].split(","))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, N = case["B"], case["N"]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=gen, device=dev) * std + mean).to(dt)

    leaves = {}
    s = {"case": case, "leaves": leaves}
    if case["op"] == "layer_norm":
        C = case["C"]
        # a residual stream: channels with offsets and scales of their own
        leaves["x"] = (torch.randn((B, N, C), generator=gen, device=dev) * (0.5 + torch.rand(C, generator=gen, device=dev)) +
                       0.3 * torch.randn(C, generator=gen, device=dev)).to(dt)
        if case["affine"]:
            leaves["weight"], leaves["bias"] = normal(C, std=0.1, mean=1.0), normal(C, std=0.1)
        if case["modulated"]:
            mod = normal(B, 6 * C, std=0.3).chunk(6, dim=1)      # what the modulation's projection returns: shift, scale and gate of two sublayers
            leaves["shift"], leaves["scale"] = mod[0], mod[1]
        s["dy"] = normal(B, N, C)
    elif case["op"] == "linear":
        K, F = case["K"], case["F"]
        leaves["x"], leaves["weight"] = normal(B, N, K), normal(F, K, std=K ** -0.5)
        if case["bias"]:
            leaves["bias"] = normal(F, std=0.1)
        if case["residual"]:
            leaves["residual"] = normal(B, N, F)
        if case["gate"]:
            leaves["gate"] = normal(B, 6 * F, std=0.5).chunk(6, dim=1)[2]
        s["dy"] = normal(B, N, F)
    else:
        H, D = case["H"], case["D"]
        shape = (B, N, H, D) if case["layout"] == "bnhd" else (B, H, N, D)
        turn = (lambda t: t.transpose(1, 2)) if case["layout"] == "bnhd" else (lambda t: t)
        leaves["x"] = turn(normal(*shape))
        s["positions"] = _places(case, gen, dev)
        s["dy"] = turn(normal(*shape))
    if case["pass"] == "train":
        for k in leaves:
            leaves[k] = leaves[k].detach().requires_grad_(True)
    else:
        del s["dy"]
    return s


# ---------------------------------------------------------------------------------------------- the plain forms, in 32 bits
def _plain_layer_norm(x, weight=None, bias=None, shift=None, scale=None):
    centred = x - x.mean(-1, keepdim=True)
    y = centred * torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    if weight is not None:
        y = y * weight + bias
    if scale is not None:
        y = y * (1 + scale[:, None]) + shift[:, None]
    return y


def _plain_linear(case, x, weight, bias=None, residual=None, gate=None):
    z = torch.matmul(x, weight.t())
    if bias is not None:
        z = z + bias
    if case["act"] == "gelu_tanh":
        z = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    elif case["act"] == "silu":
        z = z / (1 + torch.exp(-z))
    if gate is not None:
        z = z * gate[:, None]
    return z if residual is None else residual + z


def _plain_rope(case, x, positions):
    omega = [THETA ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d) for d in _axes(case)]
    angle = torch.cat([positions[..., a, None].double() * w for a, w in enumerate(omega)], -1)      # angles of far positions: 64 bits
    if angle.dim() == 3:
        angle = angle[:, None]
    sn, cs = torch.sin(angle).float(), torch.cos(angle).float()
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack([cs * even - sn * odd, sn * even + cs * odd], -1).flatten(-2)


def _plain(s, t):
    if s["case"]["op"] == "layer_norm":
        return _plain_layer_norm(**t)
    if s["case"]["op"] == "linear":
        return _plain_linear(s["case"], **t)
    return _plain_rope(s["case"], t["x"], s["positions"])


# ---------------------------------------------------------------------------------------------- the package's calls
def _package(s):
    import llsa_b200
    c, t = s["case"], s["leaves"]
    if c["op"] == "layer_norm":
        return llsa_b200.layer_norm(t["x"], t.get("weight"), t.get("bias"), EPS, scale=t.get("scale"), shift=t.get("shift"))
    if c["op"] == "linear":
        return llsa_b200.linear(t["x"], t["weight"], t.get("bias"), activation=None if c["act"] == "none" else c["act"], residual=t.get("residual"),
                                gate=t.get("gate"))
    return llsa_b200.rope_axes(t["x"], s["positions"], _axes(c), THETA)


def run(s):
    """A sampling pass returns y; a training pass y and the gradient of every input, by name."""
    train, leaves = s["case"]["pass"] == "train", s["leaves"]
    if own:
        if not train:
            with torch.no_grad():
                return {"y": _package(s)}
        y = _package(s)
        grads = torch.autograd.grad(y, list(leaves.values()), s["dy"])
        return dict(zip(["d_" + k for k in leaves], grads), y=y.detach())
    wide = {k: v.detach().float().requires_grad_(train) for k, v in leaves.items()}
    dt = leaves["x"].dtype
    if not train:
        with torch.no_grad():
            return {"y": _plain(s, wide).to(dt)}
    y = _plain(s, wide)
    grads = torch.autograd.grad(y, list(wide.values()), s["dy"].float())
    return dict(zip(["d_" + k for k in leaves], [g.to(dt) for g in grads]), y=y.detach().to(dt))


def work(case):
    """Bytes: every input (and upstream gradient) read once, every output and gradient written once.  Operations: the products of a projection,
    forward, and both gradients' where it is trained; a handful for each element elsewhere."""
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["pass"] == "train"
    rows = case["B"] * case["N"]
    if case["op"] == "layer_norm":
        n, small = rows * case["C"], (2 * case["C"] if case["affine"] else 0) + (2 * case["B"] * case["C"] if case["modulated"] else 0)
        return {"bytes": size * ((4 if train else 2) * n + (2 if train else 1) * small), "flops": (24 if train else 9) * n}
    if case["op"] == "linear":
        K, F = case["K"], case["F"]
        wide = rows * F
        small = F * K + (F if case["bias"] else 0) + (case["B"] * F if case["gate"] else 0)
        read = rows * K + small + (wide if case["residual"] else 0)
        return {"bytes": size * (read + wide + (wide + rows * K + small if train else 0)), "flops": (6 if train else 2) * rows * K * F}
    n = rows * case["H"] * case["D"]
    places = (case["B"] if case["per_sample"] else 1) * case["N"] * len(_axes(case)) * (4 if case["positions"] == "fractional" else 8)
    return {"bytes": size * (4 if train else 2) * n + places, "flops": (6 if train else 3) * n}


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_layer_norm(c, t, dy):
    x = t["x"]
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    r = 1 / torch.sqrt(var + EPS)
    h = (x - mean) * r
    w = t["weight"] if c["affine"] else torch.ones_like(x[0, 0])
    b = t["bias"] if c["affine"] else torch.zeros_like(w)
    up = 1 + t["scale"].unsqueeze(1) if c["modulated"] else torch.ones_like(x[:, :1])
    out = {"y": (h * w + b) * up + (t["shift"].unsqueeze(1) if c["modulated"] else 0)}
    if dy is None:
        return out
    g = dy * up * w
    out["d_x"] = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    if c["affine"]:
        out["d_weight"], out["d_bias"] = (dy * up * h).sum((0, 1)), (dy * up).sum((0, 1))
    if c["modulated"]:
        out["d_shift"], out["d_scale"] = dy.sum(1), (dy * (h * w + b)).sum(1)
    return out


def _exact_linear(c, t, dy):
    B, N, K, F = c["B"], c["N"], c["K"], c["F"]
    x = t["x"].reshape(B * N, K)
    z = x @ t["weight"].T
    if c["bias"]:
        z += t["bias"]
    slope = None
    if c["act"] == "gelu_tanh":      # z s(2u), u = sqrt(2 / pi) (z + 0.044715 z^3)
        s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        slope = s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
        a = z * s
    elif c["act"] == "silu":
        s = torch.sigmoid(z)
        slope, a = s * (1 + z * (1 - s)), z * s
    else:
        a = z
    a = a.reshape(B, N, F)
    y = a * t["gate"].unsqueeze(1) if c["gate"] else a
    out = {"y": y + t["residual"] if c["residual"] else y}
    if dy is None:
        return out
    dz = (dy * t["gate"].unsqueeze(1) if c["gate"] else dy).reshape(B * N, F)
    if slope is not None:
        dz = dz * slope
    out["d_x"], out["d_weight"] = (dz @ t["weight"]).reshape(B, N, K), dz.T @ x
    if c["bias"]:
        out["d_bias"] = dz.sum(0)
    if c["residual"]:
        out["d_residual"] = dy
    if c["gate"]:
        out["d_gate"] = (dy * a).sum(1)
    return out


def _exact_rope(c, t, dy, positions):
    pairs = [torch.arange(d // 2, device=positions.device, dtype=torch.float64) for d in _axes(c)]
    angle = torch.cat([positions.double()[..., a].unsqueeze(-1) * torch.exp(-(math.log(THETA) / len(i)) * i) for a, i in enumerate(pairs)], -1)
    angle = angle.unsqueeze(1) if c["per_sample"] else angle

    def turned(v, sign):
        z = torch.view_as_complex(v.contiguous().unflatten(-1, (-1, 2))) * torch.polar(torch.ones_like(angle), sign * angle)
        return torch.view_as_real(z).flatten(-2)

    return {"y": turned(t["x"], 1)} if dy is None else {"y": turned(t["x"], 1), "d_x": turned(dy, -1)}


def exact(case, seed):
    s = prepare(case, seed)
    t = {k: v.detach().double() for k, v in s["leaves"].items()}
    dy = s["dy"].double() if "dy" in s else None
    if case["op"] == "layer_norm":
        return _exact_layer_norm(case, t, dy)
    if case["op"] == "linear":
        return _exact_linear(case, t, dy)
    return _exact_rope(case, t, dy, s["positions"])
