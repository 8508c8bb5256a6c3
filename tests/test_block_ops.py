"""layer_norm, linear and rope_axes against their formulas in 64 bits.

Tolerances are counted.  u = 2^-24 is half a step of fp32; a result of type T is rounded once, which is half a step of T relative to the value (2^-24 or
2^-8).  What fp32 arithmetic adds is at most (roundings on the way) * u * (the sum of the terms' magnitudes); each test says how many.
"""
import math

import pytest
import torch

import llsa_b200

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(name, got, want, fp32_error, roundings=1.0):
    """|got - want| <= `roundings` half steps of got's type, plus what fp32 sums add."""
    tol = roundings * half_step(got.dtype) * want.abs() + fp32_error + 1e-40
    off = (got.double() - want).abs()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert bool((off <= tol).all()), "%s: off by %.3g where %.3g is allowed" % (name, float(off.max()), float(tol.flatten()[(off - tol).argmax()]))


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


# ------------------------------------------------------------------------------------------------------ layer norm
def norm_reference(x, w, b, s, t, eps, dy=None):
    """y and the gradients in 64 bits, and the magnitudes that rounding errors scale with.  x: [B, N, C]."""
    x, w, b, s, t, dy = [v.detach().double() if v is not None else None for v in (x, w, b, s, t, dy)]
    mean, mag = x.mean(-1, keepdim=True), x.abs().mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h, hb = (x - mean) * rstd, ((x - mean).abs() + mag) * rstd
    W = w if w is not None else torch.ones_like(x[0, 0])
    Bi = b if b is not None else torch.zeros_like(W)
    up = 1 + s[:, None] if s is not None else torch.ones_like(x[:, :1, :])
    sh = t[:, None] if t is not None else torch.zeros_like(x[:, :1, :])
    y, yb = (h * W + Bi) * up + sh, (hb * W.abs() + Bi.abs()) * up.abs() + sh.abs()
    if dy is None:
        return dict(y=(y, yb))
    g = dy * up * W
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    dxb = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + hb * (g.abs() * hb).mean(-1, keepdim=True))
    return dict(y=(y, yb), x=(dx, dxb), w=((dy * up * h).sum((0, 1)), (dy.abs() * up.abs() * hb).sum((0, 1))),
                b=((dy * up).sum((0, 1)), (dy.abs() * up.abs()).sum((0, 1))),
                s=((dy * (h * W + Bi)).sum(1), (dy.abs() * (hb * W.abs() + Bi.abs())).sum(1)), t=(dy.sum(1), dy.abs().sum(1)))


NORM_SHAPES = [(1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 7, 32), (2, 17, 100), (3, 33, 129), (4, 9, 384), (2, 100, 390), (1, 50, 512), (2, 31, 516), (3, 11, 1155),
               (2, 13, 2048), (1, 5, 2050), (1, 4, 4096), (2, 3, 4100), (1, 3, 5001), (1, 2, 16384), (257, 1, 48), (40, 3, 64), (2, 5000, 24)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,N,C", NORM_SHAPES)
@pytest.mark.parametrize("given", ["", "wb", "st", "wbst", "ws"])
def test_layer_norm_against_its_formula(B, N, C, dtype, given):
    g = gen(B * 1000003 + N * 1009 + C)
    eps = 1e-5
    x = normal(g, B, N, C, dtype=dtype, std=1.5, mean=0.7)
    made = dict(w=normal(g, C, dtype=dtype, std=0.2, mean=1), b=normal(g, C, dtype=dtype, std=0.2))
    mod = normal(g, B, 6 * C, dtype=dtype, std=0.3).chunk(6, 1)      # rows with a stride of their own
    made.update(s=mod[1], t=mod[4])
    p = {k: made[k].detach().requires_grad_(True) if k in given else None for k in "wbst"}
    x.requires_grad_(True)
    dy = normal(g, B, N, C, dtype=dtype)
    y = llsa_b200.layer_norm(x, p["w"], p["b"], eps, scale=p["s"], shift=p["t"])
    names = [k for k in "wbst" if k in given]
    grads = torch.autograd.grad(y, [x] + [p[k] for k in names], dy)
    ref = norm_reference(x, p["w"], p["b"], p["s"], p["t"], eps, dy)
    # 16 values of a thread, 5 steps of a warp, 32 warps: 53 additions deep, for the mean, the squares and the products; some 10 roundings beside
    within("y", y, ref["y"][0], 120 * U * ref["y"][1])
    within("dx", grads[0], ref["x"][0], 300 * U * ref["x"][1])
    for k, d in zip(names, grads[1:]):      # a sum over all rows on top
        assert d.dtype == p[k].dtype
        within("d" + k, d, ref[k][0], (200 + B * N) * U * ref[k][1])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [121, 125, 126, 127, 129, 130, 253, 254, 255, 257, 258, 381, 382, 383, 385, 386, 509, 510, 511, 513, 514, 765, 767, 769, 1019, 1021, 1022, 1023, 1025, 1026, 1027,
                               1277, 1278, 1279, 1281, 1533, 1535, 1537, 2043, 2045, 2046])
def test_layer_norm_rows_that_end_beside_a_vector(C, dtype):
    """Rows one to three channels around every multiple of what a group's vectors hold, in a tensor that begins on any of the four places beside a boundary."""
    for start in range(4):
        g = gen(7 * C + start)
        x = normal(g, start + 2 * 9 * C, dtype=dtype)[start:].view(2, 9, C)
        dy = normal(g, start + 2 * 9 * C, dtype=dtype)[start:].view(2, 9, C)
        w, b, s, t = normal(g, C), normal(g, C), normal(g, 2, C, std=0.3), normal(g, 2, C)
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b, s, t)]
        y = llsa_b200.layer_norm(*leaves[:3], 1e-5, scale=leaves[3], shift=leaves[4])
        grads = torch.autograd.grad(y, leaves, dy)
        ref = norm_reference(x, w, b, s, t, 1e-5, dy)
        within("y", y, ref["y"][0], 120 * U * ref["y"][1])
        within("dx", grads[0], ref["x"][0], 300 * U * ref["x"][1])
        for k, d in zip("wbst", grads[1:]):
            within("d" + k, d, ref[k][0], 218 * U * ref[k][1])


@pytest.mark.parametrize("param", [BF16, F32])
def test_layer_norm_takes_parameters_of_either_type(param):
    g = gen(3)
    x = normal(g, 2, 9, 96, dtype=BF16).requires_grad_(True)
    w, b = normal(g, 96, dtype=param, std=0.1, mean=1).requires_grad_(True), normal(g, 96, dtype=param).requires_grad_(True)
    s, t = normal(g, 2, 96, dtype=param, std=0.2).requires_grad_(True), normal(g, 2, 96, dtype=param).requires_grad_(True)
    dy = normal(g, 2, 9, 96, dtype=BF16)
    y = llsa_b200.layer_norm(x, w, b, 1e-5, scale=s, shift=t)
    ref = norm_reference(x, w, b, s, t, 1e-5, dy)
    within("y", y, ref["y"][0], 120 * U * ref["y"][1])
    for k, d in zip("wbst", torch.autograd.grad(y, [w, b, s, t], dy)):
        assert d.dtype == param
        within(k, d, ref[k][0], 220 * U * ref[k][1])


def test_layer_norm_any_rank_strides_and_alignment():
    g = gen(4)
    eps = 1e-6
    base = normal(g, 3, 7, 5, 48)
    want = norm_reference(base.reshape(3, 35, 48), None, None, None, None, eps)["y"]
    check = lambda y, shape: within("y", y.reshape(3, 35, 48), want[0], 120 * U * want[1])
    check(llsa_b200.layer_norm(base, eps=eps), None)
    check(llsa_b200.layer_norm(base.reshape(105, 48), eps=eps), None)
    room = torch.zeros(3, 7, 5, 60, device=DEV)
    for first in (0, 1, 3, 4):                                  # rows with gaps, on any boundary
        room[..., first:first + 48] = base
        check(llsa_b200.layer_norm(room[..., first:first + 48], eps=eps), None)
    check(llsa_b200.layer_norm(base.transpose(-1, -2).contiguous().transpose(-1, -2), eps=eps), None)      # channels apart
    token_major = base.reshape(3, 35, 48).transpose(0, 1).contiguous().transpose(0, 1)                     # [B,N,C] view of [N,B,C]
    y = llsa_b200.layer_norm(token_major, eps=eps, shift=torch.zeros(3, 48, device=DEV))
    assert y.stride() == token_major.stride()
    check(y, None)
    one = llsa_b200.layer_norm(base[0, 0, 0], eps=eps)
    assert one.shape == (48,) and torch.equal(one, llsa_b200.layer_norm(base, eps=eps)[0, 0, 0])
    shared = base[:1, :, 0].expand(3, 7, 48)                    # samples on top of one another
    assert torch.equal(llsa_b200.layer_norm(shared, eps=eps)[2], llsa_b200.layer_norm(base[:1, :, 0], eps=eps)[0])


def test_layer_norm_gradient_of_an_expanded_upstream_and_without_parameters():
    g = gen(5)
    x = normal(g, 2, 6, 40).requires_grad_(True)
    (d,) = torch.autograd.grad(llsa_b200.layer_norm(x).sum(), x)
    ref = norm_reference(x, None, None, None, None, 1e-5, torch.ones_like(x))
    within("dx", d, ref["x"][0], 300 * U * ref["x"][1])
    w = torch.ones(40, device=DEV, requires_grad=True)          # only the weight wants a gradient
    (dw,) = torch.autograd.grad(llsa_b200.layer_norm(x.detach(), w).sum(), w)
    within("dw", dw, ref["w"][0], 220 * U * ref["w"][1])


def test_layer_norm_keeps_a_bad_row_to_itself():
    g = gen(6)
    x = normal(g, 1, 8, 64, dtype=BF16)
    good = llsa_b200.layer_norm(x)
    x[0, 3, 5], x[0, 6, 1] = float("nan"), float("inf")
    y = llsa_b200.layer_norm(x)
    keep = [0, 1, 2, 4, 5, 7]
    assert torch.equal(y[0, keep], good[0, keep]) and torch.isnan(y[0, [3, 6]]).any(-1).all()
    const = llsa_b200.layer_norm(torch.full((1, 2, 64), 3.0, device=DEV), shift=torch.full((1, 64), 2.0, device=DEV))
    assert torch.equal(const, torch.full_like(const, 2.0))      # no spread: the shift alone
    far = torch.full((1, 1, 64), 1e4, device=DEV)
    far[0, 0, ::2] += 1
    assert torch.equal(llsa_b200.layer_norm(far, eps=0.0).abs(), torch.ones(1, 1, 64, device=DEV))      # a large common offset cancels nothing


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["dense", "gaps", "upstream with gaps", "one token"])
@pytest.mark.parametrize("given", ["t", "wbt", "wb", "wbst", "s"])
def test_layer_norm_gradients_have_the_same_bits_whichever_are_asked_for(given, layout, dtype):
    B, N, C = (9, 1, 130) if layout == "one token" else (3, 777, 130)
    g = gen(17)
    make = lambda gaps: normal(g, B, N + 2, C + 3, dtype=dtype)[:, 1:-1, 2:-1] if gaps else normal(g, B, N, C, dtype=dtype)
    data = dict(x=make(layout in ("gaps", "one token")), w=normal(g, C, dtype=dtype, std=0.2, mean=1), b=normal(g, C, dtype=dtype), s=normal(g, B, C, dtype=dtype, std=0.3),
                t=normal(g, B, C, dtype=dtype))
    dy = make("gaps" in layout)
    names = ["x"] + [k for k in "wbst" if k in given]
    full = {}
    for mask in reversed(range(1, 1 << len(names))):              # all of them first
        wanted = [k for i, k in enumerate(names) if mask >> i & 1]
        v = {k: data[k].detach().requires_grad_(k in wanted) for k in names}
        y = llsa_b200.layer_norm(v["x"], v.get("w"), v.get("b"), 1e-5, scale=v.get("s"), shift=v.get("t"))
        for k, d in zip(wanted, torch.autograd.grad(y, [v[k] for k in wanted], dy)):
            assert torch.equal(full.setdefault(k, d), d), (wanted, k)


# ------------------------------------------------------------------------------------------------------ projection
def act64(z, act):
    """The activation and its slope."""
    if act is None:
        return z, torch.ones_like(z)
    k = 1.0 if act == "silu" else 2 * math.sqrt(2 / math.pi)
    inner, slope = (z, torch.ones_like(z)) if act == "silu" else (z + 0.044715 * z ** 3, 1 + 3 * 0.044715 * z ** 2)
    s = torch.sigmoid(k * inner)
    return z * s, s + z * s * (1 - s) * k * slope


def linear_reference(x, w, b, act, r, gate, dy=None):
    x, w, b, r, gate, dy = [v.detach().double() if v is not None else None for v in (x, w, b, r, gate, dy)]
    K, F = w.shape[1], w.shape[0]
    z, zb = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z, zb = z + b, zb + b.abs()
    a, slope = act64(z, act)
    G = gate.reshape(gate.shape[0], *[1] * (x.dim() - 2), F) if gate is not None else 1.0
    y = a * G + (r if r is not None else 0)
    out = dict(y=y, z=z, zb=zb, G=G, slope=slope)
    if dy is not None:
        dz = (dy * G * slope)
        flat, xf = dz.reshape(-1, F), x.reshape(-1, K)
        out.update(dz=dz, x=dz @ w, xb=dz.abs() @ w.abs(), w=flat.T @ xf, wb=flat.abs().T @ xf.abs(), b=flat.sum(0), bb=flat.abs().sum(0), r=dy)
        if gate is not None:
            per = lambda t: t.reshape(gate.shape[0], -1, F).sum(1)
            out.update(g=per(dy * a), gb=per(dy.abs() * zb))
    return out


LINEAR_SHAPES = [(1, 1, 1, 1), (1, 1, 16, 16), (8, 1, 256, 384), (1, 5, 3, 7), (2, 65, 64, 64), (1, 128, 128, 192), (2, 130, 72, 200), (3, 77, 389, 133), (1, 300, 384, 3),
                 (2, 100, 390, 256), (1, 257, 520, 1032), (5, 60, 1536, 384), (2, 1000, 384, 1152), (3, 777, 384, 200), (2, 600, 64, 320), (1, 1100, 520, 72), (5, 513, 256, 136), (1, 2049, 40, 8)]
FORMS = [("plain", None, False, False), ("gelu", "gelu_tanh", False, False), ("silu", "silu", False, False), ("residual", None, True, False),
         ("gated", None, True, True), ("gelu residual", "gelu_tanh", True, False)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,N,K,F", LINEAR_SHAPES)
@pytest.mark.parametrize("form", FORMS, ids=[f[0] for f in FORMS])
def test_linear_against_its_formula(B, N, K, F, dtype, form):
    _, act, with_r, with_g = form
    g = gen(B * 1000003 + N * 1009 + K * 31 + F)
    t = dict(x=normal(g, B, N, K, dtype=dtype), w=normal(g, F, K, dtype=dtype, std=K ** -0.5), b=normal(g, F, dtype=dtype, std=0.3))
    if with_r:
        t["r"] = normal(g, B, N, F, dtype=dtype)
    if with_g:
        t["g"] = normal(g, B, 6 * F, dtype=dtype, std=0.5).chunk(6, 1)[2]
    t = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    dy = normal(g, B, N, F, dtype=dtype)
    y = llsa_b200.linear(t["x"], t["w"], t["b"], activation=act, residual=t.get("r"), gate=t.get("g"))
    grads = dict(zip(t, torch.autograd.grad(y, list(t.values()), dy)))
    check_linear(t, dy, act, y, grads, dtype)


# fp32 products of few tiles: their sums in 2, 4 and 8 parts over a cluster, forward or in dx, with ragged ends of every size
@pytest.mark.parametrize("B,N,K,F", [(2, 1000, 384, 640), (1, 1999, 660, 380), (2, 150, 389, 771), (4, 130, 1536, 384), (2, 1000, 384, 1152), (1, 70, 4099, 66)])
@pytest.mark.parametrize("form", FORMS, ids=[f[0] for f in FORMS])
def test_fp32_sums_over_a_cluster(B, N, K, F, form):
    test_linear_against_its_formula(B, N, K, F, F32, form)


def check_linear(t, dy, act, y, grads, dtype):
    M, K, F = dy.numel() // dy.shape[-1], t["x"].shape[-1], dy.shape[-1]
    ref = linear_reference(t["x"], t["w"], t.get("b"), act, t.get("r"), t.get("g"), dy)
    G = ref["G"].abs() if torch.is_tensor(ref["G"]) else 1.0
    # z: K products and additions, each within 2 u of the running sum (a tensor core cuts where an FMA rounds), and the bias.  No activation's slope
    # exceeds 1.13; the activation itself is 8 roundings, its exponential is off by 2 ulp and by u |argument| <= 80 u
    ez = (2 * K + 4) * U * ref["zb"]
    ea = 1.13 * ez + (100 * U if act else 0) * ref["z"].abs()
    r_mag = t["r"].detach().double().abs() if "r" in t else 0.0
    within("y", y, ref["y"], ea * G + 4 * U * (ref["zb"] * G + r_mag))
    # dz is rounded to its type (bf16: one half step of every term); behind an activation of bf16 data z is kept to 2^-11 of itself, and no slope changes
    # faster than 1.13 per unit of z (gelu's curvature at 0 is 2 sqrt(2 / pi) < 1.6; silu's 1/2)
    hs, adz = half_step(dtype), ref["dz"].abs()
    moved = ((2.0 ** -11 + 1e-7) if dtype == BF16 else 0.0) * ref["z"].abs() + ez + (2.0 ** -25 if dtype == BF16 else 0.0)
    edz = (1.6 * moved + 100 * U) * (dy.double().abs() * G) if act else 2 * U * adz
    keeps = act is not None or "g" in t                          # dz is written, and rounded
    edz = edz + (hs * (1 + 0.01) if keeps else 0) * (adz + edz)
    wd = t["w"].detach().double().abs()
    xf = t["x"].detach().double().abs().reshape(-1, K)
    within("dx", grads["x"], ref["x"], edz @ wd + (2 * F + 4) * U * (ref["xb"] + edz @ wd))
    flat = edz.reshape(-1, F)
    within("dw", grads["w"], ref["w"], flat.T @ xf + (2 * M + 400) * U * (ref["wb"] + flat.T @ xf))
    if "b" in grads:                                             # the sum of dz before it is rounded
        eb = ((1.6 * moved + 100 * U) * (dy.double().abs() * G) if act else 2 * U * adz).reshape(-1, F).sum(0)
        within("db", grads["b"], ref["b"], eb + (M + 100) * U * ref["bb"])
    if "r" in grads:
        assert torch.equal(grads["r"], dy)
    if "g" in grads:                                             # z is kept in the data's type: half a step of every term
        B = t["g"].shape[0]
        kept = (dy.double().abs() * (hs * 1.01 * ref["z"].abs() + ez)).reshape(B, -1, F).sum(1)
        within("dgate", grads["g"], ref["g"], kept + (M + 100) * U * ref["gb"])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_strides_ranks_and_partial_gradients(dtype):
    g = gen(11)
    K, F = 72, 40
    room = normal(g, 4, 21, 100, dtype=dtype)
    w, dy = normal(g, F, K, dtype=dtype, std=0.1), normal(g, 4, 21, F, dtype=dtype)
    for first in (0, 1, 8, 16):                                  # rows with gaps, on any boundary
        t = dict(x=room[..., first:first + K].detach().requires_grad_(True), w=w.detach().requires_grad_(True))
        y = llsa_b200.linear(t["x"], t["w"])
        check_linear(t, dy, None, y, dict(zip(t, torch.autograd.grad(y, list(t.values()), dy))), dtype)
    wt = normal(g, K, F, dtype=dtype, std=0.1).t()               # a weight stored the other way round
    t = dict(x=room[:, ::3, :K].detach().requires_grad_(True), w=wt.detach().requires_grad_(True))
    y = llsa_b200.linear(t["x"], t["w"])
    check_linear(t, dy[:, ::3], None, y, dict(zip(t, torch.autograd.grad(y, list(t.values()), dy[:, ::3]))), dtype)
    flat = llsa_b200.linear(room[0, 0, :K], w)
    assert flat.shape == (F,)
    deep = llsa_b200.linear(room[..., :K].reshape(2, 2, 3, 7, K), w)
    assert deep.shape == (2, 2, 3, 7, F) and torch.equal(deep.reshape(-1, F), llsa_b200.linear(room[..., :K].reshape(-1, K), w))
    # one gradient at a time gives the bits of all together
    full = {}
    names = ["x", "w", "b", "r", "g"]
    data = dict(x=room[..., :K], w=w, b=normal(g, F, dtype=dtype), r=normal(g, 4, 21, F, dtype=dtype), g=normal(g, 4, F, dtype=dtype))
    for wanted in [names] + [[n] for n in names]:
        t = {k: v.detach().clone().requires_grad_(k in wanted) for k, v in data.items()}
        y = llsa_b200.linear(t["x"], t["w"], t["b"], residual=t["r"], gate=t["g"])
        for k, d in zip(wanted, torch.autograd.grad(y, [t[k] for k in wanted], dy)):
            assert torch.equal(full.setdefault(k, d), d), k
    # a bias on no 16-byte boundary, a gate and a residual with gaps
    wide = normal(g, 4, 21, F + 3, dtype=dtype)
    same = llsa_b200.linear(data["x"], w, normal(gen(12), F + 1, dtype=dtype)[1:], residual=wide[..., 1:F + 1], gate=wide[:, 0, 3:])
    assert torch.equal(same, llsa_b200.linear(data["x"], w, normal(gen(12), F + 1, dtype=dtype)[1:].clone(), residual=wide[..., 1:F + 1].clone(), gate=wide[:, 0, 3:].clone()))
    # an upstream gradient that is one number everywhere
    x = room[..., :K].detach().requires_grad_(True)
    (d,) = torch.autograd.grad(llsa_b200.linear(x, w).sum(), x)
    t = dict(x=x, w=w)
    check_linear(t, torch.ones(4, 21, F, device=DEV, dtype=dtype), None, llsa_b200.linear(x, w), dict(x=d, w=linear_reference(x, w, None, None, None, None, torch.ones(4, 21, F, device=DEV))["w"]), dtype)


@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
@pytest.mark.parametrize("M,K,F,std", [(300, 64, 96, 1.0), (2000, 384, 200, 1.0), (131, 1536, 72, 3.0), (4100, 128, 200, 0.2)])
def test_slope_of_bf16_data_is_taken_from_an_fp32_product(M, K, F, std, act):
    """z is computed again and not rounded, and the bias' gradient is the sum of an unrounded dz: read in fp32 over the C ABI, it is off by fp32 roundings alone.

    The logistic s of u(z): its argument, 4 roundings, moves it by s (1 - s) |u| 4 u <= 0.9 u; 2^t is off by 2^-22 of itself, 1/4 * 4 u = 1 u; the reciprocal shared by a pair, its
    two factors and what they are made of 6 u: 8 u in all.  The slope s + z s (1 - s) u' moves by at most 1 + |z| u' for each of s, and has 8 roundings of its own."""
    import ctypes as C
    from llsa_b200 import _lib
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    g = gen(M + K)
    x, w, b, dy = normal(g, M, K, dtype=BF16), normal(g, F, K, dtype=BF16, std=std * K ** -0.5), normal(g, F, dtype=BF16, std=0.3), normal(g, M, F, dtype=BF16)
    d = dict(x=x, weight=w, bias=b, dy=dy, dx=torch.empty_like(x), dweight=torch.empty_like(w), dbias=torch.empty(F, device=DEV))
    a, keep = _lib.LlsaLinearArgs(), {k: _lib.desc(t) for k, t in d.items()}
    for k in keep:
        setattr(a, k, C.pointer(keep[k]))
    a.activation = 1 if act == "gelu_tanh" else 2
    ws = torch.empty(lib.llsa_linear_bwd_workspace_bytes(C.byref(a)) + 256, device=DEV, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = (ws.data_ptr() + 255) // 256 * 256, ws.numel() - 256
    assert lib.llsa_linear_bwd(C.byref(a), stream) == 0, lib.llsa_last_error_string()
    ref = linear_reference(x, w, b, act, None, None, dy)
    z, ez = ref["z"].abs(), (2 * K + 4) * U * ref["zb"]
    # beyond 7 (SiLU: 30) the kernel's slope stays what it is there, which is within 1e-11 of 1 or 0
    far, rise = (7.0, 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z.clamp(max=7.0) ** 2)) if act == "gelu_tanh" else (30.0, 1.0)
    edz = (1.6 * ez + 8 * U * (2 + z.clamp(max=far) * rise) + 1e-11) * dy.double().abs()
    within("db", d["dbias"], ref["b"], edz.sum(0) + (M + 100) * U * ref["bb"])
    hs = half_step(BF16)
    edz = edz + 1.01 * hs * (ref["dz"].abs() + edz)              # in front of the two products dz is rounded
    wd, xd = w.double().abs(), x.double().abs()
    within("dx", d["dx"], ref["x"], edz @ wd + (2 * F + 4) * U * (ref["xb"] + edz @ wd))
    within("dw", d["dweight"], ref["w"], edz.T @ xd + (2 * M + 400) * U * (ref["wb"] + edz.T @ xd))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_far_values(dtype):
    """Activations far out on either side, a zero gate, and rows that are not numbers."""
    z = torch.tensor([-1e30, -7e4, -300.0, -30.0, -8.0, 0.0, 8.0, 300.0, 7e4, 1e30], device=DEV)
    x = torch.zeros(1, len(z), 16, device=DEV, dtype=dtype)
    x[0, :, 0] = z.to(dtype)
    w = torch.zeros(16, 16, device=DEV, dtype=dtype)
    w[:, 0] = 1
    zz = x[0, :, 0].double()
    for act in ("gelu_tanh", "silu"):
        xg = x.detach().requires_grad_(True)
        y = llsa_b200.linear(xg, w, activation=act)
        arg = zz if act == "silu" else 2 * math.sqrt(2 / math.pi) * (zz + 0.044715 * zz ** 3)
        s = torch.sigmoid(arg)
        # e^-t with t off by 3 roundings, 3 u |t|, is off by that much relative to itself; below e^-100 nothing of an fp32 result is left
        rel = 2 * half_step(dtype) + 4 * U * arg.abs().clamp(max=100)
        assert ((y[0, :, 3].double() - zz * s).abs() <= rel * (zz * s).abs() + 1e-30).all(), act
        (d,) = torch.autograd.grad(y[..., 3].sum(), xg)
        _, slope = act64(zz.clamp(-1e4, 1e4), act)
        assert torch.isfinite(d).all() and ((d[0, :, 0].double() - slope).abs() <= 4 * half_step(dtype) * slope.abs() + 1e-6).all(), act
    g = gen(12)
    x, w, r = normal(g, 1, 9, 64, dtype=dtype), normal(g, 24, 64, dtype=dtype), normal(g, 1, 9, 24, dtype=dtype)
    closed = torch.zeros(1, 24, device=DEV, dtype=dtype).requires_grad_(True)
    y = llsa_b200.linear(x, w, residual=r, gate=closed)
    assert torch.equal(y, r)                                      # as a freshly initialised adaLN-zero block leaves its input
    (d,) = torch.autograd.grad(y.sum(), closed)
    assert (d != 0).all()
    good = llsa_b200.linear(x, w)
    x[0, 4, 7] = float("nan")
    bad = llsa_b200.linear(x, w)
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.isnan(bad[0, 4]).all() and torch.equal(bad[0, keep], good[0, keep])


# ------------------------------------------------------------------------------------------------------ rotary positions
def rope_reference(x, pos, axes, theta, sign=1.0):
    x = x.detach().double()
    ang = torch.cat([pos[..., a, None].double() * theta ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d) for a, d in enumerate(axes)], -1)
    ang = sign * (ang[:, None] if ang.dim() == 3 else ang)
    e, o = x[..., 0::2], x[..., 1::2]
    y = torch.stack([ang.cos() * e - ang.sin() * o, ang.sin() * e + ang.cos() * o], -1).flatten(-2)
    mag = torch.stack([e.abs() + o.abs()] * 2, -1).flatten(-2)
    return y, mag


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,N,axes", [(1, 1, 1, (2,)), (1, 2, 3, (2, 4)), (2, 3, 65, (32, 32)), (1, 6, 100, (16, 24, 24)), (3, 5, 33, (10,)), (2, 4, 17, (6, 6, 2, 4)),
                                        (4, 6, 257, (64, 64)), (1, 1, 5000, (64,)), (2, 1, 7, (256, 256))])
@pytest.mark.parametrize("kind", ["int64", "int32", "float32", "per sample"])
def test_rope_axes_against_its_formula(B, H, N, axes, dtype, kind):
    g = gen(B + 7 * H + 31 * N + sum(axes))
    x = normal(g, B, N, H, sum(axes), dtype=dtype).transpose(1, 2).requires_grad_(True)      # heads side by side, as a projection leaves them
    shape = (B, N, len(axes)) if kind == "per sample" else (N, len(axes))
    pos = torch.randint(-1000, 1 << 20, shape, generator=g, device=DEV)
    if kind == "int32":
        pos = pos.int()
    if kind == "float32":
        pos = pos.float() * 0.01
    y = llsa_b200.rope_axes(x, pos, axes, 10000.0)
    assert y.stride() == x.stride()
    dy = normal(g, B, H, N, sum(axes), dtype=dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    # the angle in units of pi is rounded to fp32 once (pi u / 2), sine and cosine are off by 2 ulp, and three more roundings: below 8 u
    for got, (want, mag) in ((y, rope_reference(x, pos, axes, 10000.0)), (dx, rope_reference(dy, pos, axes, 10000.0, -1.0))):
        within("rope", got, want, 8 * U * mag)


def test_rope_axes_strides_alignment_and_table():
    g = gen(21)
    pos = torch.randint(0, 64, (40, 2), generator=g, device=DEV)
    room = normal(g, 2, 3, 40, 80, dtype=BF16)
    want = llsa_b200.rope_axes(room[..., :64].contiguous(), pos, (32, 32))
    for first in (0, 1, 2, 8):
        room2 = torch.zeros(2, 3, 40, 80, device=DEV, dtype=BF16)
        room2[..., first:first + 64] = room[..., :64]
        assert torch.equal(llsa_b200.rope_axes(room2[..., first:first + 64], pos, (32, 32)), want)
    apart = room[..., :64].transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(llsa_b200.rope_axes(apart, pos, (32, 32)), want)
    shared = room[:, :1, :, :64].expand(2, 3, 40, 64)
    assert torch.equal(llsa_b200.rope_axes(shared, pos, (32, 32))[:, 2], want[:, 0])
    assert torch.equal(llsa_b200.rope_axes(room[..., :64], pos.repeat(1, 2)[:, :2], (32, 32)), want)           # positions with a row stride
    assert torch.equal(llsa_b200.rope_axes(room[..., :64], pos.t().contiguous().t(), (32, 32)), want)          # and axis by axis
    # my_rope_fn with an fp32 table of the same angles: equal up to the table's rounding and the order of the arithmetic
    x = normal(g, 1, 2, 40, 64)
    om = 10000.0 ** (-torch.arange(0, 32, 2, device=DEV, dtype=torch.float64) / 32)
    ang = torch.cat([pos[:, a, None].double() * om for a in range(2)], -1)
    table = torch.stack([ang.sin(), ang.cos()], -1).flatten(-2).float()
    _, mag = rope_reference(x, pos, (32, 32), 10000.0)
    assert ((llsa_b200.rope_axes(x, pos, (32, 32)) - llsa_b200.my_rope_fn(x, table)).double().abs() <= 12 * U * mag).all()


def test_rope_axes_turns_back_and_differentiates_twice():
    g = gen(22)
    x = normal(g, 1, 2, 9, 32).requires_grad_(True)
    pos = torch.arange(9, device=DEV)[:, None]
    y = llsa_b200.rope_axes(x, pos, (32,))
    dy = normal(g, 1, 2, 9, 32).requires_grad_(True)
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dx, dy, x.detach())              # the rotation again
    assert torch.equal(ddy, y)


# ------------------------------------------------------------------------------------------------------ differences, streams, graphs, compiler
@pytest.mark.parametrize("what", ["norm", "linear gelu", "linear gated", "rope"])
def test_gradients_against_differences(what):
    """The kernel's gradient along a direction against central differences of the formula in 64 bits.  The step of 1e-4 leaves an error of
    about 1e-8 of the third derivative; fp32 gradients carry some 1e-6."""
    g = gen(31)
    if what == "norm":
        leaves = [normal(g, 2, 5, 33), normal(g, 33, mean=1.0, std=0.2), normal(g, 33), normal(g, 2, 33, std=0.3), normal(g, 2, 33)]
        f = lambda x, w, b, s, t: llsa_b200.layer_norm(x, w, b, 1e-3, scale=s, shift=t)
        ref = lambda x, w, b, s, t: norm_reference(x, w, b, s, t, 1e-3)["y"][0]
    elif what == "linear gelu":
        leaves = [normal(g, 2, 5, 20), normal(g, 11, 20, std=0.3), normal(g, 11)]
        f = lambda x, w, b: llsa_b200.linear(x, w, b, activation="gelu_tanh")
        ref = lambda x, w, b: linear_reference(x, w, b, "gelu_tanh", None, None)["y"]
    elif what == "linear gated":
        leaves = [normal(g, 2, 5, 20), normal(g, 11, 20, std=0.3), normal(g, 11), normal(g, 2, 5, 11), normal(g, 2, 11)]
        f = lambda x, w, b, r, gt: llsa_b200.linear(x, w, b, residual=r, gate=gt)
        ref = lambda x, w, b, r, gt: linear_reference(x, w, b, None, r, gt)["y"]
    else:
        leaves, pos = [normal(g, 2, 3, 5, 12)], torch.randint(0, 50, (5, 2), generator=g, device=DEV)
        f = lambda x: llsa_b200.rope_axes(x, pos, (4, 8))
        ref = lambda x: rope_reference(x, pos, (4, 8), 10000.0)[0]
    leaves = [t.requires_grad_(True) for t in leaves]
    y = f(*leaves)
    dy = normal(g, *y.shape)
    grads = torch.autograd.grad(y, leaves, dy)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = normal(g, *leaf.shape).double()
        at = lambda e: (ref(*[t.detach().double() + (e * v if j == i else 0) for j, t in enumerate(leaves)]) * dy.double()).sum()
        want = float((at(1e-4) - at(-1e-4)) / 2e-4)
        got = float((grad.double() * v).sum())
        scale = float((grad.double() * v).abs().sum())
        assert abs(got - want) <= 2e-5 * scale + 1e-6, (what, i, got, want)


def _block(x, w1, b1, w2, mod, pos):
    """One run of the operators together, as a block calls them."""
    shift, scale, gate = mod.chunk(3, 1)
    B, N, C = x.shape
    h = llsa_b200.layer_norm(x, eps=1e-6, scale=scale, shift=shift)
    h = llsa_b200.rope_axes(h.view(B, N, 2, C // 2).transpose(1, 2), pos, (C // 4, C // 4)).transpose(1, 2).reshape(B, N, C)
    return llsa_b200.linear(llsa_b200.linear(h, w1, b1, activation="gelu_tanh"), w2, residual=x, gate=gate)


def _block_leaves(seed, dtype=BF16, B=2, N=150, C=128):
    g = gen(seed)
    leaves = [normal(g, B, N, C, dtype=dtype), normal(g, 4 * C, C, dtype=dtype, std=C ** -0.5), normal(g, 4 * C, dtype=dtype),
              normal(g, C, 4 * C, dtype=dtype, std=C ** -0.5 / 2), normal(g, B, 3 * C, dtype=dtype, std=0.4)]
    return leaves, normal(g, B, N, C, dtype=dtype), torch.stack([torch.arange(N, device=DEV) // 16, torch.arange(N, device=DEV) % 16], -1)


def _pass(leaves, dy, pos):
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    y = _block(*leaves, pos)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def test_operators_together_against_64_bits():
    leaves, dy, pos = _block_leaves(41)
    wide = [t.double().requires_grad_(True) for t in leaves]
    x, w1, b1, w2, mod = wide
    shift, scale, gate = mod.chunk(3, 1)
    B, N, C = x.shape
    mean = x.mean(-1, keepdim=True)
    h = (x - mean) / ((x - mean).square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + scale[:, None]) + shift[:, None]
    om = 10000.0 ** (-torch.arange(0, C // 4, 2, device=DEV, dtype=torch.float64) / (C // 4))
    ang = torch.cat([pos[:, a, None].double() * om for a in range(2)], -1)
    hh = h.view(B, N, 2, C // 2).transpose(1, 2)
    e, o = hh[..., 0::2], hh[..., 1::2]
    h = torch.stack([ang.cos() * e - ang.sin() * o, ang.sin() * e + ang.cos() * o], -1).flatten(-2).transpose(1, 2).reshape(B, N, C)
    z = h @ w1.T + b1
    y = x + gate[:, None] * ((z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))) @ w2.T)
    want = [y.detach(), *torch.autograd.grad(y, wide, dy.double())]
    # four values rounded to bf16 on the way forward and six on the way back, each 2^-8 of itself at most and independent: in the norm at most 10 of them
    for name, a, b in zip(["y", "dx", "dw1", "db1", "dw2", "dmod"], _pass(leaves, dy, pos), want):
        assert float((a.double() - b).norm()) <= 10 * 2.0 ** -8 * float(b.norm()), name


def test_same_bits_every_time_on_any_stream_and_in_graphs():
    sets = [_block_leaves(s) for s in (51, 52)]
    want = [_pass(*s) for s in sets]
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(_pass(*s), w))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(3):                                            # two streams at once
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = _pass(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [None, None]
    ins = [[t.clone() for t in sets[0][0]], [t.clone() for t in sets[0][0]]]
    for i in range(2):                                            # two captured graphs, replayed on other inputs, at the same time
        with torch.cuda.graph(graphs[i]):
            outs[i] = _pass(ins[i], sets[0][1], sets[0][2])
    for i in range(2):
        for t, v in zip(ins[i], sets[i][0]):
            t.copy_(v)
    w1 = _pass(sets[1][0], sets[0][1], sets[0][2])
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[0], want[0])) and all(torch.equal(p, q) for p, q in zip(outs[1], w1))


def test_first_call_of_a_thread():
    """A thread that has made no CUDA call yet, as the autograd engine's before its first backward: tensor maps need a context there."""
    import threading
    leaves, dy, pos = _block_leaves(63)
    want = _pass(leaves, dy, pos)
    t, w = torch.randn(64, 64, device=DEV).bfloat16(), torch.randn(64, 64, device=DEV).bfloat16()
    one = llsa_b200.linear(t, w)
    torch.cuda.synchronize()
    got = {}

    def work():
        try:
            got["one"] = llsa_b200.linear(t, w)
            got["pass"] = _pass(leaves, dy, pos)
            torch.cuda.synchronize()
        except Exception as e:      # shown by the assertion below
            got["error"] = e

    th = threading.Thread(target=work)
    th.start()
    th.join()
    assert "error" not in got, got["error"]
    assert torch.equal(got["one"], one) and all(torch.equal(a, b) for a, b in zip(got["pass"], want))


def test_operators_trace():
    leaves, dy, pos = _block_leaves(61)
    want = _pass(leaves, dy, pos)
    fn = torch.compile(_block, backend="aot_eager", fullgraph=True)
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    y = fn(*leaves, pos)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nothing_to_do(dtype):
    """No rows: empty results, and gradients of the parameters that are zero."""
    w, b = torch.ones(24, 16, device=DEV, dtype=dtype, requires_grad=True), torch.ones(24, device=DEV, dtype=dtype, requires_grad=True)
    for shape in ((0, 5, 16), (3, 0, 16)):
        x = torch.zeros(shape, device=DEV, dtype=dtype, requires_grad=True)
        s = torch.ones(shape[0], 16, device=DEV, dtype=dtype, requires_grad=True)
        lw = torch.ones(16, device=DEV, dtype=dtype, requires_grad=True)
        y = llsa_b200.layer_norm(x, lw, None, scale=s)
        assert y.shape == shape
        for d in torch.autograd.grad(y.sum(), [lw, s]):
            assert not d.any()
        gate = torch.ones(shape[0], 24, device=DEV, dtype=dtype, requires_grad=True)
        y = llsa_b200.linear(x, w, b, residual=torch.zeros(*shape[:2], 24, device=DEV, dtype=dtype), gate=gate)
        assert y.shape == (*shape[:2], 24)
        for d, t in zip(torch.autograd.grad(y.sum(), [x, w, b, gate]), (x, w, b, gate)):
            assert d.shape == t.shape and not d.any()
    x = torch.zeros(2, 0, 5, 16, device=DEV, dtype=dtype)
    assert llsa_b200.rope_axes(x, torch.zeros(5, 1, device=DEV), (16,)).shape == x.shape


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act,gated", [(0, False), (1, False), (0, True)])
def test_c_backward_without_rows_clears_the_parameters_gradients(dtype, act, gated):
    import ctypes as C
    from llsa_b200 import _lib
    K, F = 32, 48
    room = torch.zeros(1, 64, device=DEV, dtype=dtype)            # rows that begin somewhere
    outs = dict(dweight=torch.full((F, K), 7.0, device=DEV, dtype=dtype), dbias=torch.full((F,), 7.0, device=DEV, dtype=dtype))
    given = dict(x=room[:0, :K], weight=torch.ones(F, K, device=DEV, dtype=dtype), dy=room[:0, :F], dx=room[:0, :K], **outs)
    if gated:
        given.update(gate=torch.ones(3, F, device=DEV, dtype=dtype), dgate=torch.full((3, F), 7.0, device=DEV, dtype=dtype))
        outs["dgate"] = given["dgate"]
    a, keep = _lib.LlsaLinearArgs(), {}
    for name, t in given.items():
        keep[name] = _lib.desc(t)
        keep[name].ptr = keep[name].ptr or room.data_ptr()        # torch gives an empty tensor no address
        setattr(a, name, C.pointer(keep[name]))
    a.activation = act
    assert _lib.lib().llsa_linear_bwd_workspace_bytes(C.byref(a)) == 0
    assert _lib.lib().llsa_linear_bwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0, _lib.lib().llsa_last_error_string()
    for name, t in outs.items():
        assert not t.any(), name


def test_refusals():
    x, w = torch.zeros(2, 4, 16, device=DEV), torch.zeros(8, 16, device=DEV)
    r, gate = torch.zeros(2, 4, 8, device=DEV), torch.zeros(2, 8, device=DEV)
    pos = torch.zeros(4, 1, device=DEV)
    x4 = torch.zeros(1, 2, 4, 16, device=DEV)
    for exc, call in [
        (TypeError, lambda: llsa_b200.linear(x.half(), w.half())), (TypeError, lambda: llsa_b200.linear(x, w.bfloat16())),
        (TypeError, lambda: llsa_b200.linear(x, w, residual=r.bfloat16())), (TypeError, lambda: llsa_b200.layer_norm(x.half())),
        (TypeError, lambda: llsa_b200.layer_norm(x, torch.ones(16, device=DEV, dtype=BF16))), (TypeError, lambda: llsa_b200.rope_axes(x4, pos.double(), (16,))),
        (ValueError, lambda: llsa_b200.linear(x, w, activation="relu")),
        (RuntimeError, lambda: llsa_b200.linear(x, w.t())), (RuntimeError, lambda: llsa_b200.linear(x, w, torch.zeros(16, device=DEV))),
        (RuntimeError, lambda: llsa_b200.linear(x, w, residual=r[:1])), (RuntimeError, lambda: llsa_b200.linear(x, w, gate=gate)),
        (RuntimeError, lambda: llsa_b200.linear(x, w, activation="silu", residual=r, gate=gate)), (RuntimeError, lambda: llsa_b200.linear(x, w, residual=r, gate=gate[:1])),
        (RuntimeError, lambda: llsa_b200.linear(x, w.cpu())), (RuntimeError, lambda: llsa_b200.layer_norm(x, torch.ones(15, device=DEV))),
        (RuntimeError, lambda: llsa_b200.layer_norm(x, scale=torch.ones(1, 16, device=DEV))), (RuntimeError, lambda: llsa_b200.layer_norm(x, eps=float("nan"))),
        (RuntimeError, lambda: llsa_b200.layer_norm(x, eps=-1.0)), (RuntimeError, lambda: llsa_b200.layer_norm(torch.zeros(1, 16385, device=DEV))),
        (RuntimeError, lambda: llsa_b200.layer_norm(x, torch.ones(16))), (RuntimeError, lambda: llsa_b200.rope_axes(x4, pos, (8, 8))),
        (RuntimeError, lambda: llsa_b200.rope_axes(x4, pos, (14,))), (RuntimeError, lambda: llsa_b200.rope_axes(x4, pos[:3], (16,))),
        (RuntimeError, lambda: llsa_b200.rope_axes(x4, pos.repeat(1, 2), (15, 1))), (RuntimeError, lambda: llsa_b200.rope_axes(x4, pos, (16,), theta=0.0)),
        (RuntimeError, lambda: llsa_b200.rope_axes(x4, pos.requires_grad_(True), (16,))), (RuntimeError, lambda: llsa_b200.rope_axes(x, pos, (16,))),
    ]:
        with pytest.raises(exc):
            call()
    xg = x.requires_grad_(True)                                   # what cannot be differentiated again says so
    (d,) = torch.autograd.grad(llsa_b200.linear(xg, w, activation="silu").sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError):
        llsa_b200.layer_norm(fwd.make_dual(x.detach(), torch.ones_like(x)))


# ------------------------------------------------------------------------------------------------------ unusual calls
def test_a_bad_value_stays_where_the_formula_puts_it():
    """NaN in one row of the weight, in the bias, in one row of x: what does not depend on it is what it is without."""
    g = gen(71)
    x, w, b = normal(g, 2, 300, 64, dtype=BF16), normal(g, 72, 64, dtype=BF16, std=0.2), normal(g, 72, dtype=BF16)
    dy = normal(g, 2, 300, 72, dtype=BF16)
    for act in ("gelu_tanh", "silu"):
        def grads(x, w, b):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
            y = llsa_b200.linear(leaves[0], leaves[1], leaves[2], activation=act)
            return y.detach(), *torch.autograd.grad(y, leaves, dy)
        want = grads(x, w, b)
        for f in (0, 7, 40, 71):
            others = [i for i in range(72) if i != f]
            for bad_w in (True, False):
                w2, b2 = w.clone(), b.clone()
                if bad_w:
                    w2[f, 3] = float("nan")
                else:
                    b2[f] = float("nan")
                y, dx, dw, db = grads(x, w2, b2)
                assert y[..., f].isnan().all() and dw[f].isnan().all() and db[f].isnan() and dx.isnan().all()
                assert torch.equal(y[..., others], want[0][..., others]) and torch.equal(dw[others], want[2][others]) and torch.equal(db[others], want[3][others])
        x2 = x.clone()
        x2[1, 77, 5] = float("nan")
        y, dx, dw, db = grads(x2, w, b)
        assert y[1, 77].isnan().all() and dx[1, 77].isnan().all() and dw.isnan().all() and db.isnan().all()
        y[1, 77], dx[1, 77] = want[0][1, 77], want[1][1, 77]
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [9, 128, 200, 256, 300])
@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
def test_an_infinite_weight_keeps_to_the_rows_that_are_there(M, act, dtype):
    """Rows of a tile behind the last one have no product, not 0 times infinity: far out an activation's slope is 1 or 0, and so is that of an infinite z."""
    g = gen(72)
    x, w, b, dy = normal(g, M, 64, dtype=dtype).abs() + 1, normal(g, 72, 64, dtype=dtype, std=0.2), normal(g, 72, dtype=dtype), normal(g, M, 72, dtype=dtype)
    up, down = [0, 40], [7, 71]
    others = [f for f in range(72) if f not in up + down]

    def grads(w):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = llsa_b200.linear(*leaves, activation=act)
        return y.detach(), *torch.autograd.grad(y, leaves[1:], dy)

    _, dw, db = grads(w)
    w2 = w.clone()
    w2[up, 3], w2[down, 3] = float("inf"), float("-inf")
    y2, dw2, db2 = grads(w2)
    assert torch.equal(dw2[others], dw[others]) and torch.equal(db2[others], db[others])
    assert (y2[:, up] == float("inf")).all()
    d64, x64 = dy.double(), x.double()
    within("db", db2[up], d64[:, up].sum(0), (M + 100) * U * d64[:, up].abs().sum(0))
    # dz of slope 1 is dy, to a rounding of the slope in fp32 that may take it a half step of dy's type off
    within("dw", dw2[up], d64[:, up].T @ x64, (2 * M * U + half_step(dtype)) * (d64[:, up].abs().T @ x64))
    # slope 0: s(-7) of GELU is below 1e-15, s(-30) of SiLU times 30 below 3e-12
    assert float(db2[down].abs().max()) <= 3e-12 * float(d64.abs().sum(0).max()) and float(dw2[down].abs().max()) <= 3e-12 * float((d64.abs().T @ x64).max())


def _long_samples(seed, B=3, N=1030, K=96, F=136):
    g = gen(seed)
    leaves = [normal(g, B, N, K, dtype=BF16), normal(g, F, K, dtype=BF16, std=K ** -0.5), normal(g, F, dtype=BF16, std=0.1), normal(g, B, N, F, dtype=BF16),
              normal(g, B, F, dtype=BF16)]
    return [t.requires_grad_(True) for t in leaves], normal(g, B, N, F, dtype=BF16)


def _gated(x, w, b, r, gate):
    return llsa_b200.linear(x, w, b, residual=r, gate=gate)


@pytest.mark.parametrize("B,N,K,F", [(3, 1030, 96, 136), (1, 4096, 64, 72), (5, 520, 256, 64)])
def test_gradient_of_a_gate_of_long_samples_does_without_the_product(B, N, K, F):
    """No z is kept and rounded: dgate in fp32 over the C ABI is a sum over the features of sums over the rows, 2 N + 2 K roundings deep and some 100 of their joining."""
    import ctypes as C
    from llsa_b200 import _lib
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    (x, w, b, r, gate), dy = _long_samples(83, B, N, K, F)
    x, w, b, gate = [t.detach() for t in (x, w, b, gate)]
    d = dict(x=x.view(B * N, K), weight=w, bias=b, gate=gate, dy=dy.view(B * N, F), dgate=torch.empty(B, F, device=DEV), dbias=torch.empty(F, device=DEV))
    a, keep = _lib.LlsaLinearArgs(), {k: _lib.desc(t) for k, t in d.items()}
    for k in keep:
        setattr(a, k, C.pointer(keep[k]))
    assert lib.llsa_linear_keeps_product(C.byref(a)) == 0
    ws = torch.empty(lib.llsa_linear_bwd_workspace_bytes(C.byref(a)) + 256, device=DEV, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = (ws.data_ptr() + 255) // 256 * 256, ws.numel() - 256
    assert lib.llsa_linear_bwd(C.byref(a), stream) == 0, lib.llsa_last_error_string()
    ref = linear_reference(x, w, b, None, None, gate, dy)
    within("dgate", d["dgate"], ref["g"], (2 * N + 2 * K + 100) * U * ref["gb"])
    within("db", d["dbias"], ref["b"], (B * N + 100) * U * ref["bb"])


def test_gate_of_long_samples_in_parts_in_graphs_and_traced():
    """Any of the gradients alone has the bits that it has among all of them; so it has captured, replayed and traced."""
    leaves, dy = _long_samples(81)
    want = torch.autograd.grad(_gated(*leaves), leaves, dy)
    for mask in range(1, 32):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(leaves)]
        wanted = [i for i in range(5) if mask >> i & 1]
        got = torch.autograd.grad(_gated(*some), [some[i] for i in wanted], dy)
        for i, d in zip(wanted, got):
            assert torch.equal(d, want[i]), (mask, i)
    other, dy2 = _long_samples(82)
    want2 = torch.autograd.grad(_gated(*other), other, dy2)
    ins, dyc = [t.detach().clone().requires_grad_(True) for t in leaves], dy.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_gated(*ins), ins, dyc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = torch.autograd.grad(_gated(*ins), ins, dyc)
    for src, d, expect in ((leaves, dy, want), (other, dy2, want2), (leaves, dy, want)):
        with torch.no_grad():
            for t, v in zip(ins, src):
                t.copy_(v)
            dyc.copy_(d)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, expect))
    y = torch.compile(_gated, backend="aot_eager", fullgraph=True)(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


# a gate of long samples; of short ones; products, slope, both tiles of one CTA and of a pair
@pytest.mark.parametrize("M,K,F,act,gate", [(4096, 384, 1536, "gelu_tanh", 0), (4096, 1536, 384, None, 2), (300, 100, 72, "silu", 0), (1200, 256, 512, None, 12),
                                            (128, 64, 64, None, 0), (16384, 64, 64, "silu", 0)])
@pytest.mark.parametrize("limit", [1, 2, 8, 32])
def test_every_value_behind_an_expired_wait_is_nan(M, K, F, act, gate, limit, monkeypatch):
    """Under a poll limit of a few looks results are final or NaN, the status word says so under set_device_checks, and the next call is right."""
    from llsa_b200 import ops
    g = gen(M + K + F)
    x, w, b = normal(g, gate or 1, M // (gate or 1), K, dtype=BF16), normal(g, F, K, dtype=BF16, std=K ** -0.5), normal(g, F, dtype=BF16)
    r, gt, dy = normal(g, *x.shape[:2], F, dtype=BF16), normal(g, gate, F, dtype=BF16) if gate else None, normal(g, *x.shape[:2], F, dtype=BF16)
    leaves = [t.requires_grad_(True) for t in (x, w, b, gt) if t is not None]

    def run():
        y = llsa_b200.linear(x, w, b, activation=act, residual=r if gate else None, gate=gt)
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    want = run()
    for t in run():                                               # so that what a limited call finds in memory is not the answer
        t.fill_(3.0)
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_wait_limit", limit)
    ops._native()
    got = run()
    torch.cuda.synchronize()
    try:
        llsa_b200.set_device_checks(True)
        ops._native()
        if limit == 1:
            with pytest.raises(RuntimeError, match="bounded wait"):
                llsa_b200.linear(x, w, b)
    finally:
        monkeypatch.setattr(ops, "_wait_limit", 0)
        llsa_b200.set_device_checks(False)
        ops._native()
    for a, c in zip(got, want):
        assert bool((a.isnan() | (a == c)).all()), int((~a.isnan() & (a != c)).sum())
    if limit == 1:
        assert got[0].isnan().any()
    assert all(torch.equal(a, c) for a, c in zip(run(), want))


def test_broadcast_operands_and_inference_mode():
    """Expanded inputs count once for every place they stand in, and their gradients are summed back; inference tensors go through."""
    g = gen(101)
    x, w = normal(g, 40, 64, dtype=BF16).requires_grad_(True), normal(g, 48, 64, dtype=BF16, std=0.2).requires_grad_(True)
    row = normal(g, 48, dtype=BF16).requires_grad_(True)
    mod = normal(g, 64).requires_grad_(True)
    one = normal(g, 1, dtype=BF16).requires_grad_(True)
    dy = normal(g, 3, 40, 48, dtype=BF16)

    def wide(x, w, row, mod, one):
        h = llsa_b200.layer_norm(x.expand(3, 40, 64), one.expand(64), scale=mod.expand(3, 64), shift=mod.expand(3, 64))
        return llsa_b200.linear(h, w, one.expand(48), residual=row.expand(3, 40, 48), gate=row.expand(3, 48))

    def dense(x, w, row, mod, one):
        c = lambda t, *shape: t.expand(*shape).contiguous()
        h = llsa_b200.layer_norm(c(x, 3, 40, 64), c(one, 64), scale=c(mod, 3, 64), shift=c(mod, 3, 64))
        return llsa_b200.linear(h, w, c(one, 48), residual=c(row, 3, 40, 48), gate=c(row, 3, 48))

    leaves = [x, w, row, mod, one]
    a, b = wide(*leaves), dense(*leaves)
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, leaves, dy), torch.autograd.grad(b, leaves, dy)):
        assert torch.equal(p, q)
    with torch.inference_mode():
        y = wide(*[t.detach() for t in leaves])
        z = llsa_b200.rope_axes(y.view(3, 1, 40, 48), torch.arange(40, device=DEV)[:, None], (48,))
    assert torch.equal(y, a) and torch.isfinite(z).all()
    assert torch.equal(llsa_b200.linear(x[0], w), llsa_b200.linear(x[:1], w)[0]) and torch.equal(llsa_b200.layer_norm(x[0]), llsa_b200.layer_norm(x[:1])[0])


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows have the bits that a call of them alone has, and no others."""
    g = gen(91)
    M, C = 2_200_000, 1024
    x = torch.empty(M, C, device=DEV, dtype=BF16)
    tail = normal(g, 1000, C, dtype=BF16)
    x.zero_()[-1000:] = tail
    w, b = normal(g, C, dtype=BF16), normal(g, C, dtype=BF16)
    y = llsa_b200.layer_norm(x, w, b)
    assert torch.equal(y[-1000:], llsa_b200.layer_norm(tail, w, b)) and torch.equal(y[:5], b.expand(5, C))
    xg, wg = x.requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(llsa_b200.layer_norm(xg, wg, b), (xg, wg), y)
    tg = tail.clone().requires_grad_(True)
    (dt,) = torch.autograd.grad(llsa_b200.layer_norm(tg, w, b), tg, y[-1000:].contiguous())
    zg = torch.zeros(5, C, device=DEV, dtype=BF16, requires_grad=True)
    (d0,) = torch.autograd.grad(llsa_b200.layer_norm(zg, w, b), zg, y[:5].contiguous())
    assert torch.equal(dx[-1000:], dt) and torch.equal(dx[:5], d0) and torch.isfinite(dw).all()
    del dx, y, xg
    x = x.detach()
    rows = x.view(1, M // 1000, 1000, C)
    pos = torch.arange(1000, device=DEV)[:, None]
    turned = llsa_b200.rope_axes(rows[..., :512], pos, (512,))
    assert torch.equal(turned[:, -1:], llsa_b200.rope_axes(rows[:, -1:, :, :512], pos, (512,))) and not turned[:, 0].any()
    del turned, rows
    w1, b1 = normal(g, 1024, 64, dtype=BF16), normal(g, 1024, dtype=BF16)
    small = x[:, :64]                                             # rows 2 KB apart
    y = llsa_b200.linear(small, w1, b1, activation="silu")
    near = llsa_b200.linear(tail[:, :64], w1, b1, activation="silu")
    zero = llsa_b200.linear(torch.zeros(8, 64, device=DEV, dtype=BF16), w1, b1, activation="silu")
    assert torch.equal(y[-1000:], near) and torch.equal(y[:8], zero)
    xg, wg = small.requires_grad_(True), w1.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(llsa_b200.linear(xg, wg, b1, activation="silu"), (xg, wg), y)
    tg = tail[:, :64].clone().requires_grad_(True)
    wt = w1.clone().requires_grad_(True)
    dt, dwt = torch.autograd.grad(llsa_b200.linear(tg, wt, b1, activation="silu"), (tg, wt), near)
    # dx of a row: sums over 1024 features, of the same bf16 terms, in fp32: 1024 roundings of what may stand in any order, and one to bf16
    mag = (near.double().abs() * 2) @ w1.double().abs()
    within("dx", dx[-1000:], dt.double(), 2 * 1024 * U * mag, 2.0)
    # rows of zeros add nothing to dw; what is left are sums over 1000 rows
    mag = (near.double().abs() * 2).t() @ tail[:, :64].double().abs()
    within("dw", dw, dwt.double(), 2 * 1000 * U * mag, 2.0)


def test_outputs_of_the_c_entries_leave_their_surroundings_alone():
    """Rows of y, dx and z inside larger matrices: nothing between or behind them is written."""
    import ctypes as C
    from llsa_b200 import _lib
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for dtype in (BF16, F32):
        for M, K, F in ((130, 64, 72), (257, 40, 200), (1, 8, 8), (300, 64, 66)):
            g = gen(M + F)
            x, w, dy = normal(g, M, K, dtype=dtype), normal(g, F, K, dtype=dtype), normal(g, M, F, dtype=dtype)
            want = llsa_b200.linear(x, w)
            for pad in (8, 16, 3):
                big = torch.full((M + 4, F + pad), 7.0, device=DEV, dtype=dtype)
                a = _lib.LlsaLinearArgs()
                keep = [_lib.desc(t) for t in (x, w, big[2:-2, :F])]
                a.x, a.weight, a.y = [C.pointer(d) for d in keep]
                assert lib.llsa_linear_fwd(C.byref(a), stream) == 0, lib.llsa_last_error_string()
                assert torch.equal(big[2:-2, :F], want), (dtype, M, K, F, pad)
                big[2:-2, :F] = 7.0
                assert bool((big == 7.0).all())
                big = torch.full((M + 4, K + pad), 7.0, device=DEV, dtype=dtype)
                b = _lib.LlsaLinearArgs()
                keep = [_lib.desc(t) for t in (x, w, dy, big[2:-2, :K])]
                b.x, b.weight, b.dy, b.dx = [C.pointer(d) for d in keep]
                ws = torch.empty(max(1, lib.llsa_linear_bwd_workspace_bytes(C.byref(b))) + 256, device=DEV, dtype=torch.uint8)
                b.workspace, b.workspace_bytes = (ws.data_ptr() + 255) // 256 * 256, ws.numel() - 256
                assert lib.llsa_linear_bwd(C.byref(b), stream) == 0, lib.llsa_last_error_string()
                xg = x.clone().requires_grad_(True)
                (dx,) = torch.autograd.grad(llsa_b200.linear(xg, w), xg, dy)
                assert torch.equal(big[2:-2, :K], dx), (dtype, M, K, F, pad)
                big[2:-2, :K] = 7.0
                assert bool((big == 7.0).all())
        for B, N, Ch in ((2, 9, 64), (3, 5, 130), (1, 4, 384)):
            x = normal(gen(Ch), B, N, Ch, dtype=dtype)
            for pad in (4, 8, 3):
                big = torch.full((B + 2, N + 2, Ch + pad), 7.0, device=DEV, dtype=dtype)
                out = big[1:-1, 1:-1, :Ch]
                keep = [_lib.desc(x), _lib.desc(out)]
                assert lib.llsa_layer_norm_fwd(C.byref(keep[0]), None, None, None, None, 1e-5, C.byref(keep[1]), None, stream) == 0, lib.llsa_last_error_string()
                want = norm_reference(x, None, None, None, None, 1e-5)["y"]
                within("y", out, want[0], (Ch + 16) * U * want[1])
                out.fill_(7.0)
                assert bool((big == 7.0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act,gated", [(0, False), (1, False), (0, True)])
def test_c_entries_take_a_residual_and_an_upstream_gradient_of_rows_that_overlap(dtype, act, gated):
    """One row for all, and a window that moves by eight: the bits of the same rows written out."""
    import ctypes as C
    from llsa_b200 import _lib
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    M, K, F = 300, 64, 72
    g = gen(19)
    x, w, gate, line = normal(g, M, K, dtype=dtype), normal(g, F, K, dtype=dtype, std=0.1), normal(g, 3, F, dtype=dtype), normal(g, 8 * M + F, dtype=dtype)

    def call(rows):
        d = dict(x=x, weight=w, residual=rows, y=torch.empty(M, F, device=DEV, dtype=dtype), dy=rows, dx=torch.empty(M, K, device=DEV, dtype=dtype),
                 dweight=torch.empty(F, K, device=DEV, dtype=dtype), dbias=torch.empty(F, device=DEV, dtype=dtype))
        if gated:
            d.update(gate=gate, pre=torch.empty(M, F, device=DEV, dtype=dtype), dgate=torch.empty(3, F, device=DEV, dtype=dtype))
        elif act and dtype == F32:
            d.update(pre=torch.empty(M, F, device=DEV, dtype=dtype))
        a, keep = _lib.LlsaLinearArgs(), {k: _lib.desc(t) for k, t in d.items()}
        for k in keep:
            setattr(a, k, C.pointer(keep[k]))
        a.activation = act
        assert lib.llsa_linear_fwd(C.byref(a), stream) == 0, lib.llsa_last_error_string()
        ws = torch.empty(max(1, lib.llsa_linear_bwd_workspace_bytes(C.byref(a))) + 256, device=DEV, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = (ws.data_ptr() + 255) // 256 * 256, ws.numel() - 256
        assert lib.llsa_linear_bwd(C.byref(a), stream) == 0, lib.llsa_last_error_string()
        torch.cuda.synchronize()
        return [d[k] for k in ("y", "dx", "dweight", "dbias") + (("dgate",) if gated else ())]

    for step in (0, 8):
        rows = line.as_strided((M, F), (step, 1))
        for k, p, q in zip(("y", "dx", "dweight", "dbias", "dgate"), call(rows), call(rows.contiguous())):
            if k in ("dbias", "dgate"):                          # a thread owns one column or eight neighbours: the same terms, below `most`, in another order, rounded on either side
                most = float(rows.abs().max()) * max(1.13, float(gate.abs().max()), float((x.float().abs() @ w.float().abs().T).max()))
                assert bool(((p.double() - q.double()).abs() <= 2.02 * half_step(dtype) * q.double().abs() + 2 * (M + 100) * U * M * most).all()), k
            else:
                assert torch.equal(p, q), k


# ------------------------------------------------------------------------------------------------------ the model
@pytest.mark.parametrize("attn,fused_rope,side", [("sparse_l2", True, 128), ("sparse_l1", False, 32), ("pixel", True, 16)])
def test_model_on_the_fused_block_agrees_with_the_eager_block(attn, fused_rope, side):
    from llsa_b200.dit import RopeDiT
    torch.manual_seed(1)
    a = RopeDiT(layers=2, sample_size=side, attn_type=attn, fused_rope=fused_rope).to(DEV)
    b = RopeDiT(layers=2, sample_size=side, attn_type=attn, fused_rope=fused_rope, fused_block=True).to(DEV)
    b.load_state_dict(a.state_dict())
    x, t = torch.randn(2, 3, side, side, device=DEV), torch.tensor([321, 7], device=DEV)
    out = []
    for m in (a, b):
        with torch.autocast("cuda", dtype=BF16):
            y = m(x, t)
        y.float().square().mean().backward()
        out.append(y)
    # two bf16 evaluations of one model whose selections may differ in a few blocks
    assert out[0].shape == out[1].shape and float((out[0].float() - out[1].float()).norm()) <= 3e-2 * float(out[0].float().norm())
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert torch.isfinite(q.grad).all(), n
        assert float((p.grad - q.grad).norm()) <= 0.1 * float(p.grad.norm()) + 1e-12, n


def test_model_on_the_fused_block_in_fp32():
    from llsa_b200.dit import RopeDiT
    torch.manual_seed(2)
    a = RopeDiT(heads=2, layers=2, sample_size=16, attn_type="pixel").to(DEV)
    b = RopeDiT(heads=2, layers=2, sample_size=16, attn_type="pixel", fused_block=True).to(DEV)
    b.load_state_dict(a.state_dict())
    x, t = torch.randn(2, 3, 16, 16, device=DEV), torch.tensor([321, 7], device=DEV)
    ya, yb = a(x, t), b(x, t)
    ya.square().mean().backward()
    yb.square().mean().backward()
    assert float((ya - yb).norm()) <= 1e-5 * float(ya.norm())
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert float((p.grad - q.grad).norm()) <= 1e-4 * float(p.grad.norm()) + 1e-12, n
