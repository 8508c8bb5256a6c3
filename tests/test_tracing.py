"""The layer operators under torch.compile and the checks of torch.library: traced whole, shape functions as the kernels allocate."""
import subprocess
import sys

import pytest
import torch

import llsa_b200
from llsa_b200 import ops, synth

DEV = "cuda:0"

# a fresh process: the first call of the library is the traced one
_FIRST_CALL = """
import torch, llsa_b200
from llsa_b200 import synth
q, k, v, do = [t.cuda() for t in synth.gaussian_qkv(1, 1, 2, 4096, 64, dtype=torch.bfloat16)]
table = torch.ones(4096, 64, device="cuda", dtype=torch.bfloat16)
w = torch.ones(64, device="cuda", requires_grad=True)
for call in (lambda *x: llsa_b200.llsa_l2(*x), lambda *x: llsa_b200.llsa_l1_rope(*x, table), lambda *x: llsa_b200.llsa_l2_rms_rope(*x, w, w, table)):
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = torch.compile(lambda *x: call(*x) * 2, fullgraph=True, backend="aot_eager")(*x)
    want = call(*x) * 2
    assert torch.equal(o, want)
    got, want = [torch.autograd.grad(t, x, do) for t in (o, want)]
    # dq and dv repeat exactly or up to the order of fp32 sums in front of a rounding to bf16
    assert all(float((a.float() - b.float()).norm() / b.float().norm()) < 1e-3 for a, b in zip(got, want))
"""


@pytest.mark.gpu
def test_whole_graph_compile_of_a_first_call():
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]


def _operands(layout, N=2048, dtype=torch.bfloat16):
    q, k, v, do = [t.to(DEV) for t in synth.gaussian_qkv(1, 1, 2, N, 64, dtype=dtype)]
    if layout == "bnhd":
        q, k, v, do = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    if layout == "expanded":
        k, v = [t[:, :1].expand(1, 2, N, 64) for t in (k, v)]
    if layout == "offset":                            # rows that no kernel takes as they are
        q = torch.cat([q, q], -1)[..., 8:72]
    return [t.detach().requires_grad_(True) for t in (q, k, v)] + [do]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "expanded", "offset"])
def test_operators_as_torch_library_checks_them(layout):
    """Shape functions, schemas (no output shares memory with another or with an input) and autograd registration."""
    ops._ready()
    L = torch.ops.llsa_b200
    q, k, v, do = _operands(layout)
    table, w = torch.ones(2048, 64, device=DEV, dtype=q.dtype), torch.ones(64, device=DEV, requires_grad=True)
    for front, two in (((None, None, None, 0.0), 0), ((None, None, None, 0.0), 8), ((table, w, w, 1e-5), 0)):
        torch.library.opcheck(L.layer_fwd.default, (q, k, v, *front, 8, two, 16, 2 if two else 1),
                              test_utils=("test_schema", "test_faketensor", "test_autograd_registration", "test_aot_dispatch_static"))
    q, k, v, w = [t.detach() for t in (q, k, v, w)]
    which = ("test_schema", "test_faketensor")
    o, saved, qr, kr = L.layer_fwd(q, k, v, table, w, w, 1e-5, 8, 0, 16, 1)
    torch.library.opcheck(L.layer_bwd.default, (do, qr, kr, v, o, saved, table, q, k, w, w, 1e-5, 8, 0, 16, 1, True), test_utils=which)
    one, two = llsa_b200.llsa_l1_debug(q, k, v, 8, 16), llsa_b200.llsa_l2_debug(q, k, v, 8, 8, 16)
    for dbg, low, lists in ((one, (None, None), (None, 8, 0)), (two, (two["pk2"], two["pv2"]), (two["p_indices"], 8, 8))):
        args = (q, k, v, dbg["pk"], dbg["pv"], *low)
        torch.library.opcheck(L.attn_fwd.default, args + (dbg["indices"], *lists, 16, 16.0, 256.0), test_utils=which)
        torch.library.opcheck(L.attn_bwd.default, (do, *args, dbg["o"], dbg["lse"], dbg["indices"], *lists, 16, 16.0, 256.0, 16.0, 256.0, False),
                              test_utils=which)


# Layouts of x [2, 6, 40, 64] or of three dimensions: dense, channels apart, permuted with dense channels, rows with gaps, samples and rows on top of one another
_LAYOUTS = {
    "dense": lambda m: m(2, 6, 40, 64),
    "channels apart": lambda m: m(2, 6, 64, 40).transpose(2, 3),
    "tokens in front": lambda m: m(2, 40, 6, 64).transpose(1, 2),
    "everything permuted": lambda m: m(64, 40, 6, 2).permute(3, 2, 1, 0),
    "gaps": lambda m: m(2, 6, 40, 80)[..., 3:67],
    "rows on top of one another": lambda m: m(2, 6, 1, 64).expand(2, 6, 40, 64),
    "samples on top of one another": lambda m: m(1, 6, 40, 64).expand(2, 6, 40, 64),
    "one number everywhere": lambda m: m(1, 1, 1, 1).expand(2, 6, 40, 64),
    "three, dense": lambda m: m(2, 40, 64),
    "three, channels apart": lambda m: m(2, 64, 40).transpose(1, 2),
    "three, tokens in front": lambda m: m(40, 2, 64).transpose(0, 1),
    "two, channels apart": lambda m: m(64, 40).t(),
    "one channel": lambda m: m(2, 40, 6, 1).transpose(1, 2),
}
# y's strides, where y is not laid out as empty_like(x) says: the kernels read a dense copy
_DENSE = {"channels apart", "everything permuted", "gaps", "rows on top of one another", "samples on top of one another", "one number everywhere",
          "three, channels apart", "two, channels apart"}
# (four dimensions that do not follow one another)
_DENSE_NORM = _DENSE | {"tokens in front", "one channel"}


def _strides(shape):
    out = [1]
    for n in reversed(shape[1:]):
        out.insert(0, out[0] * n)
    return tuple(out)


@pytest.mark.parametrize("layout", _LAYOUTS)
def test_traced_results_are_laid_out_as_the_kernels_lay_them_out(layout):
    """Strides that the shape functions give, against the rule: y as x is, where its channels are dense, else contiguous."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops._native()
    with FakeTensorMode():
        x = _LAYOUTS[layout](lambda *shape: torch.empty(shape, device="cuda"))
        y = torch.ops.llsa_b200.layer_norm_fwd(x, None, None, None, None, 1e-5, True)[0]
        assert y.shape == x.shape and y.stride() == (_strides(x.shape) if layout in _DENSE_NORM else x.stride())
        if x.dim() == 4 and x.shape[-1] > 1:
            y = torch.ops.llsa_b200.rope_axes(x, torch.empty(40, 1, device="cuda"), (64,), 1e4, False)
            assert y.shape == x.shape and y.stride() == (_strides(x.shape) if layout in _DENSE else x.stride())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", _LAYOUTS)
def test_traced_layouts_are_the_real_ones(layout, dtype):
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops._ready()
    L = torch.ops.llsa_b200
    x = _LAYOUTS[layout](lambda *shape: torch.randn(shape, device=DEV, dtype=dtype))
    pos = torch.arange(40, device=DEV)[:, None]
    calls = [lambda x, pos: L.layer_norm_fwd(x, None, None, None, None, 1e-5, False), lambda x, pos: L.layer_norm_fwd(x, None, None, None, None, 1e-5, True)]
    if x.dim() == 4 and x.shape[-1] > 1:
        calls.append(lambda x, pos: [L.rope_axes(x, pos, (64,), 1e4, False)])
    for call in calls:
        real = call(x, pos)
        with FakeTensorMode() as mode:
            traced = call(mode.from_tensor(x), mode.from_tensor(pos))
        assert [(t.shape, t.stride(), t.dtype) for t in traced] == [(t.shape, t.stride(), t.dtype) for t in real]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_operators_as_torch_library_checks_them(dtype):
    ops._ready()
    L = torch.ops.llsa_b200
    which, both = ("test_schema", "test_faketensor"), ("test_schema", "test_faketensor", "test_autograd_registration", "test_aot_dispatch_static")
    g = torch.Generator(device=DEV).manual_seed(5)
    r = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(dtype)
    for C in (64, 61):
        x, w, b, s, t = r(2, 40, C), r(C), r(C), r(2, C), r(2, C)
        for xx in (x, r(2, C, 40).transpose(1, 2), r(2, 5, 8, C + 3)[..., 3:]):
            torch.library.opcheck(L.layer_norm_fwd.default, tuple(v.detach().requires_grad_(True) for v in (xx, w, b, s, t)) + (1e-5, False), test_utils=both)
        stats = L.layer_norm_fwd(x, w, b, s, t, 1e-5, True)[1]
        for want in (0, 3, 15):
            torch.library.opcheck(L.layer_norm_bwd.default, (r(2, 40, C), x, w, b, s, stats, want, dtype, dtype), test_utils=which)
    for K, F, N in ((64, 48, 40), (61, 47, 40), (64, 48, 600)):
        x, w, b, res, gate, dy = r(2, N, K), r(F, K), r(F), r(2, N, F), r(2, F), r(2, N, F)
        for act, rr, gg in ((0, None, None), (1, None, None), (2, res, None), (0, res, gate)):
            leaves = [v.detach().requires_grad_(True) if v is not None else None for v in (x, w, b, rr, gg)]
            torch.library.opcheck(L.linear_fwd.default, (*leaves, act, False, False), test_utils=both)
            torch.library.opcheck(L.linear_fwd.default, (x, w, b, rr, gg, act, gg is not None or (act > 0 and dtype == torch.float32), True), test_utils=which)
            pre = L.linear_fwd(x, w, b, rr, gg, act, True, False)[1]
            torch.library.opcheck(L.linear_bwd.default, (dy, x, w, b, pre, gg, None, None, act, 15 if gg is not None else 7), test_utils=which)
    pos = torch.arange(40, device=DEV)[:, None]
    for x in (r(2, 3, 40, 64), r(2, 40, 3, 64).transpose(1, 2), r(2, 3, 64, 40).transpose(2, 3)):
        torch.library.opcheck(L.rope_axes.default, (x.detach().requires_grad_(True), pos, (64,), 1e4, False), test_utils=both)


@pytest.mark.gpu
def test_model_without_permutation_traces():
    """Its first layer norm reads the transposed view that the convolution leaves."""
    from llsa_b200.dit import RopeDiT
    torch.manual_seed(3)
    m = RopeDiT(heads=2, layers=1, sample_size=16, attn_type="pixel", token_permutation=False, fused_block=True).to(DEV)
    x, t = torch.randn(2, 3, 16, 16, device=DEV), torch.tensor([321, 7], device=DEV)
    with torch.no_grad():
        want = m(x, t)
        got = torch.compile(m, backend="aot_eager", fullgraph=True)(x, t)
    # the projection in front is a convolution of torch's either way, in fp32
    assert float((got - want).norm()) <= 1e-4 * float(want.norm())
