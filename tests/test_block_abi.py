"""What the C entries of layer_norm, linear and rope_axes refuse before anything reaches a GPU, and what they answer from sizes alone."""
import ctypes as C
import os
import shutil
import subprocess
import sys

import pytest
import torch

from llsa_b200 import _lib
from test_cabi import ERR_ARG, ERR_DTYPE, ERR_NULL, ERR_SHAPE, ERR_STRIDE, ERR_WORKSPACE, HEADER, OK, fake

BF16, F32 = torch.bfloat16, torch.float32
ref = C.byref


def linear_args(M=64, K=32, F=48, dtype=BF16, act=0, **given):
    """The arguments of a call, and their descriptors, which have to outlive it; given: descriptors by field, None to leave one out."""
    d = dict(x=fake((M, K), dtype), weight=fake((F, K), dtype), y=fake((M, F), dtype))
    d.update(given)
    a = _lib.LlsaLinearArgs()
    for name, t in d.items():
        if t is not None:
            setattr(a, name, C.pointer(t))
    a.activation = act
    return a, d


def test_struct_layout_matches_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = [name for name, _ in _lib.LlsaLinearArgs._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "llsa_b200.h"\nint main(void) {\n  printf("%zu\\n", sizeof(LlsaLinearArgs));\n' +
                   "".join('  printf("%s %%zu\\n", offsetof(LlsaLinearArgs, %s));\n' % (f, f) for f in fields) + "  return 0;\n}\n")
    subprocess.run([cc, "-I", os.path.dirname(HEADER), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    assert int(out[0]) == C.sizeof(_lib.LlsaLinearArgs)
    for line in out[1:]:
        if line.strip():
            name, off = line.split()
            assert getattr(_lib.LlsaLinearArgs, name).offset == int(off), name


@pytest.mark.parametrize("code,change", [
    (ERR_NULL, dict(x=None)), (ERR_NULL, dict(weight=None)), (ERR_NULL, dict(y=None)), (ERR_NULL, dict(x=fake((64, 32), ptr=None))),
    (ERR_DTYPE, dict(x=fake((64, 32), torch.int32))), (ERR_DTYPE, dict(weight=fake((48, 32), F32))), (ERR_DTYPE, dict(y=fake((64, 48), F32))),
    (ERR_DTYPE, dict(bias=fake((48,), F32))), (ERR_DTYPE, dict(residual=fake((64, 48), F32))),
    (ERR_SHAPE, dict(x=fake((64, 1, 32)))), (ERR_SHAPE, dict(weight=fake((48, 40)))), (ERR_SHAPE, dict(y=fake((63, 48)))), (ERR_SHAPE, dict(bias=fake((47,)))),
    (ERR_SHAPE, dict(residual=fake((64, 47)))), (ERR_SHAPE, dict(residual=fake((64, 48)), gate=fake((5, 48)))), (ERR_SHAPE, dict(residual=fake((64, 48)), gate=fake((0, 48)))),
    (ERR_SHAPE, dict(x=fake((64, 0)), weight=fake((48, 0)))),
    (ERR_STRIDE, dict(x=fake((64, 32), strides=(64, 2)))), (ERR_STRIDE, dict(x=fake((64, 32), strides=(36, 1)))), (ERR_STRIDE, dict(x=fake((64, 32), ptr=0x10002))),
    (ERR_STRIDE, dict(weight=fake((48, 32), ptr=0x10008))), (ERR_STRIDE, dict(y=fake((64, 48), strides=(1, 64)))), (ERR_STRIDE, dict(bias=fake((48,), strides=(2,)))),
    (ERR_ARG, dict(act=3)), (ERR_ARG, dict(act=-1)), (ERR_ARG, dict(gate=fake((2, 48)))), (ERR_ARG, dict(act=1, residual=fake((64, 48)), gate=fake((2, 48)))),
    (ERR_ARG, dict(pre=fake((64, 48)))),
])
def test_linear_forward_refuses(code, change):
    a, keep = linear_args(**change)
    assert _lib.lib().llsa_linear_fwd(ref(a), None) == code, _lib.lib().llsa_last_error_string()
    assert _lib.lib().llsa_last_error_string()


def test_linear_without_rows_does_nothing():
    a, keep = linear_args(M=0)
    assert _lib.lib().llsa_linear_fwd(ref(a), None) == OK
    assert _lib.lib().llsa_linear_fwd(None, None) == ERR_NULL


@pytest.mark.parametrize("code,change", [
    (ERR_NULL, dict(dy=None)), (ERR_SHAPE, dict(dy=fake((64, 47)))), (ERR_DTYPE, dict(dy=fake((64, 48), F32))), (ERR_STRIDE, dict(dy=fake((64, 48), strides=(1, 64)))),
    (ERR_SHAPE, dict(dx=fake((64, 48)))), (ERR_DTYPE, dict(dx=fake((64, 32), F32))), (ERR_STRIDE, dict(dweight=fake((48, 32), strides=(40, 1)))),
    (ERR_DTYPE, dict(dweight=fake((48, 32), F32))), (ERR_SHAPE, dict(dbias=fake((47,)))), (ERR_DTYPE, dict(dbias=fake((48,), torch.int32))),
    (ERR_NULL, dict(dgate=fake((2, 48)), pre=fake((64, 48)))), (ERR_NULL, dict(gate=fake((2, 48)), dgate=fake((2, 48)))),
    (ERR_SHAPE, dict(gate=fake((2, 48)), dgate=fake((1, 48)), pre=fake((64, 48)))),
    (ERR_NULL, dict(dtype=F32, act=1, dy=fake((64, 48), F32), dx=fake((64, 32), F32))),
])
def test_linear_backward_refuses(code, change):
    a, keep = linear_args(**{**dict(y=None, dy=fake((64, 48))), **change})
    lib = _lib.lib()
    need = lib.llsa_linear_bwd_workspace_bytes(ref(a))
    a.workspace, a.workspace_bytes = 0x100000, max(need, 0)
    assert lib.llsa_linear_bwd(ref(a), None) == code, lib.llsa_last_error_string()


@pytest.mark.parametrize("dtype,act,gated", [(F32, 1, False), (F32, 0, True), (BF16, 0, True)])
def test_linear_refuses_a_kept_product_off_its_boundary(dtype, act, gated):
    """The pass over dy reads 16 bytes of dy and of the kept product at once: `contiguous` includes a base on a 16-byte boundary, in either direction."""
    lib = _lib.lib()
    step = 4 if dtype == F32 else 2
    mk = lambda *shape, **k: fake(shape, dtype, **k)
    for off, code in ((step, ERR_STRIDE), (8, ERR_STRIDE), (16 - step, ERR_STRIDE)):
        given = dict(x=mk(64, 32), weight=mk(48, 32), pre=mk(64, 48, ptr=0x10000 + off))
        if gated:
            given.update(gate=mk(2, 48), residual=mk(64, 48))
        a, keep = linear_args(dtype=dtype, act=act, **given)
        assert lib.llsa_linear_fwd(ref(a), None) == code and b"pre" in lib.llsa_last_error_string()
        given.update(y=None, residual=None, dy=mk(64, 48), dx=mk(64, 32))
        a, keep = linear_args(dtype=dtype, act=act, **given)
        a.workspace, a.workspace_bytes = 0x100000, 1 << 30
        assert lib.llsa_linear_bwd_workspace_bytes(ref(a)) == -1
        assert lib.llsa_linear_bwd(ref(a), None) == code and b"pre" in lib.llsa_last_error_string()


def test_linear_backward_wants_its_workspace():
    lib = _lib.lib()
    a, keep = linear_args(y=None, dy=fake((64, 48)), dx=fake((64, 32)), dweight=fake((48, 32)), dbias=fake((48,)), act=1)
    need = lib.llsa_linear_bwd_workspace_bytes(ref(a))
    assert need > 64 * 48 * 2
    for ws, size in ((None, need), (0x100000, need - 1), (0x100010, need)):
        a.workspace, a.workspace_bytes = ws, size
        assert lib.llsa_linear_bwd(ref(a), None) == ERR_WORKSPACE
    bad, keep2 = linear_args(weight=fake((48, 40)))
    assert lib.llsa_linear_bwd_workspace_bytes(ref(bad)) == -1 and lib.llsa_linear_keeps_product(ref(bad)) == -1


@pytest.mark.parametrize("change", [dict(x=fake((64, 32), strides=(0, 1))), dict(x=fake((64, 32), strides=(16, 1))), dict(weight=fake((48, 32), strides=(0, 1))),
                                    dict(weight=fake((48, 32), strides=(24, 1)))])
def test_linear_refuses_rows_that_overlap(change):
    """bf16 operands of the products: tensor maps are specified for strides that reach past a row.  One row has no stride."""
    lib = _lib.lib()
    a, keep = linear_args(**change)
    assert lib.llsa_linear_fwd(ref(a), None) == ERR_STRIDE and b"overlap" in lib.llsa_last_error_string()
    assert lib.llsa_linear_keeps_product(ref(a)) == -1 and lib.llsa_linear_bwd_workspace_bytes(ref(a)) == -1
    a, keep = linear_args(M=1, x=fake((1, 32), strides=(0, 1)))
    assert lib.llsa_linear_keeps_product(ref(a)) == 0
    long = dict(x=fake((1024, 32)), dy=fake((1024, 48), strides=(0, 1)), gate=fake((2, 48)), dx=fake((1024, 32)))      # a gate of long samples
    a, keep = linear_args(M=1024, y=None, **long)
    a.workspace, a.workspace_bytes = 0x100000, max(0, lib.llsa_linear_bwd_workspace_bytes(ref(a)))
    assert lib.llsa_linear_bwd(ref(a), None) == ERR_STRIDE and b"dy" in lib.llsa_last_error_string()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act,gated", [(0, False), (1, False), (2, False), (0, True)])
def test_linear_backward_without_rows_wants_no_workspace(dtype, act, gated):
    """In a process of its own: what goes wrong in a plan for no rows may end it."""
    code = '''
import ctypes as C, torch
from test_block_abi import _lib, fake, linear_args
F = 48
given = dict(y=None, x=fake((0, 32), {0}), weight=fake((F, 32), {0}), dy=fake((0, F), {0}), dx=fake((0, 32), {0}))
if {2}:
    given["gate"] = fake((3, F), {0})
a, keep = linear_args(M=0, F=F, dtype={0}, act={1}, **given)
lib = _lib.lib()
assert lib.llsa_linear_bwd_workspace_bytes(C.byref(a)) == 0
assert lib.llsa_linear_bwd(C.byref(a), None) == 0, lib.llsa_last_error_string()
'''.format(dtype, act, gated)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(__file__),
                       env=dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))])))
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


# long samples, and one step beside each side of the rule
@pytest.mark.parametrize("B,N,K,F,dtype", [(2, 512, 256, 64, BF16), (2, 511, 64, 64, BF16), (2, 512, 264, 64, BF16), (1, 1024, 512, 8, BF16), (3, 600, 100, 64, BF16),
                                           (3, 600, 96, 60, BF16), (2, 1024, 64, 64, F32), (1, 64, 16, 16, BF16), (65535, 512, 8, 8, BF16), (65536, 512, 8, 8, BF16)])
@pytest.mark.parametrize("gated", [True, False])
def test_kept_product_is_what_tracing_expects(B, N, K, F, dtype, gated):
    """The traced forward's results have the sizes that the library's rule gives them."""
    from llsa_b200 import ops
    from torch._subclasses.fake_tensor import FakeTensorMode
    pad = (K + 7) // 8 * 8
    a, keep = linear_args(M=B * N, K=K, F=F, x=fake_rows(B * N, K, pad, dtype), weight=fake_rows(F, K, pad, dtype), y=None, gate=fake_rows(B, F, F, dtype) if gated else None)
    keeps = _lib.lib().llsa_linear_keeps_product(ref(a))
    assert keeps >= 0, _lib.lib().llsa_last_error_string()
    if not gated:
        assert keeps == 0
        return
    assert keeps == (0 if dtype == BF16 and N >= 512 and N >= 2 * K and K % 8 == 0 and F % 8 == 0 and B <= 65535 else 1)
    ops._native()
    with FakeTensorMode():
        x, w = torch.empty(B, N, K, dtype=dtype, device="cuda"), torch.empty(F, K, dtype=dtype, device="cuda")
        r, g = torch.empty(B, N, F, dtype=dtype, device="cuda"), torch.empty(B, F, dtype=dtype, device="cuda")
        out = torch.ops.llsa_b200.linear_fwd(x, w, None, r, g, 0, True, False)
    assert out[0].shape == (B, N, F) and out[1].shape == (B * N if keeps else 0, F)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act,gated", [(0, False), (1, False), (2, False), (0, True)])
@pytest.mark.parametrize("N", [40, 600, 0])
def test_traced_forward_keeps_the_product_where_the_library_does(dtype, act, gated, N):
    """Asked to keep it, whatever stands behind the product."""
    from llsa_b200 import ops
    from torch._subclasses.fake_tensor import FakeTensorMode
    B, K, F = 2, 64, 48
    a, keep = linear_args(M=B * N, K=K, F=F, x=fake_rows(B * N, K, K, dtype), weight=fake_rows(F, K, K, dtype), y=None, act=act,
                          gate=fake_rows(B, F, F, dtype) if gated else None)
    keeps = _lib.lib().llsa_linear_keeps_product(ref(a))
    assert keeps >= 0, _lib.lib().llsa_last_error_string()
    ops._native()
    with FakeTensorMode():
        x, w = torch.empty(B, N, K, dtype=dtype, device="cuda"), torch.empty(F, K, dtype=dtype, device="cuda")
        r, g = torch.empty(B, N, F, dtype=dtype, device="cuda"), torch.empty(B, F, dtype=dtype, device="cuda")
        out = torch.ops.llsa_b200.linear_fwd(x, w, None, r if gated else None, g if gated else None, act, True, False)
    assert out[1].shape == (B * N if keeps else 0, F)


def fake_rows(rows, cols, ld, dtype):
    """A descriptor of [rows, cols] with rows `ld` apart, of memory that is nowhere."""
    d = fake((1, cols), dtype)
    d.shape[0], d.shape[1], d.stride[0], d.stride[1] = rows, cols, ld, 1
    return d


def norm_call(x=None, w=None, b=None, s=None, t=None, eps=1e-5, y=None, stats=None):
    keep = [x if x is not None else fake((2, 10, 64)), w, b, s, t, y if y is not None else fake((2, 10, 64)), stats]
    p = [ref(k) if k is not None else None for k in keep]
    return _lib.lib().llsa_layer_norm_fwd(p[0], p[1], p[2], p[3], p[4], eps, p[5], p[6], None)


def test_layer_norm_forward_refuses():
    lib = _lib.lib()
    assert lib.llsa_layer_norm_fwd(None, None, None, None, None, 1e-5, None, None, None) == ERR_NULL
    assert norm_call(x=fake((2, 10, 64), torch.int32)) == ERR_DTYPE
    assert norm_call(y=fake((2, 10, 64), F32)) == ERR_DTYPE
    assert norm_call(w=fake((64,), torch.int32)) == ERR_DTYPE
    assert norm_call(x=fake((2, 10, 64), F32), y=fake((2, 10, 64), F32), s=fake((2, 64))) == ERR_DTYPE      # bf16 beside fp32 data
    assert norm_call(x=fake((20, 64))) == ERR_SHAPE
    assert norm_call(x=fake((1, 1, 16385)), y=fake((1, 1, 16385))) == ERR_SHAPE
    assert norm_call(y=fake((2, 10, 63))) == ERR_SHAPE
    assert norm_call(w=fake((63,))) == ERR_SHAPE and norm_call(s=fake((3, 64))) == ERR_SHAPE and norm_call(t=fake((64,))) == ERR_SHAPE
    assert norm_call(stats=fake((2, 10, 3), F32)) == ERR_SHAPE
    assert norm_call(x=fake((2, 10, 64), strides=(10 * 128, 128, 2))) == ERR_STRIDE
    assert norm_call(s=fake((2, 64), strides=(128, 2))) == ERR_STRIDE
    for eps in (-1e-6, float("nan")):
        assert norm_call(eps=eps) == ERR_ARG
    assert norm_call(x=fake((0, 10, 64)), y=fake((0, 10, 64))) == OK


def test_layer_norm_backward_refuses():
    lib = _lib.lib()
    x, dy, dx, st = fake((2, 10, 64)), fake((2, 10, 64)), fake((2, 10, 64)), fake((2, 10, 2), F32)
    s, dw, ds = fake((2, 64)), fake((64,)), fake((2, 64))
    n = lib.llsa_layer_norm_bwd_partial_elems(2, 10, 64, 1)
    part, short = fake((n,), F32), fake((n - 1,), F32)

    def call(x=x, dy=dy, scale=s, stats=st, dx=dx, dw=None, ds=None, part=None):
        p = [ref(k) if k is not None else None for k in (dy, x, None, None, scale, stats, dx, dw, None, ds, None, part)]
        return lib.llsa_layer_norm_bwd(*p, None)

    assert call(x=None) == ERR_NULL and call(dy=None) == ERR_NULL and call(dx=None) == ERR_NULL and call(stats=None) == ERR_NULL
    assert call(dw=dw) == ERR_NULL                                # the partial sums have no room
    assert call(dw=dw, part=short) == ERR_WORKSPACE and call(ds=ds, part=fake((n,))) == ERR_WORKSPACE
    assert call(dy=fake((2, 10, 64), F32)) == ERR_DTYPE and call(stats=fake((2, 10, 2))) == ERR_DTYPE and call(dw=fake((64,), torch.int32), part=part) == ERR_DTYPE
    assert call(dy=fake((2, 9, 64))) == ERR_SHAPE and call(ds=fake((1, 64)), part=part) == ERR_SHAPE
    assert call(ds=fake((2, 64), strides=(128, 1)), part=part) == ERR_STRIDE
    assert call(scale=None, dy=fake((2, 10, 64), strides=(11 * 64, 64, 1))) == ERR_STRIDE      # nothing is per sample: rows follow one another
    assert lib.llsa_layer_norm_bwd_partial_elems(0, 10, 64, 1) == 0 and lib.llsa_layer_norm_bwd_partial_elems(2, 10, 16385, 1) == 0


def test_rope_axes_refuses():
    lib = _lib.lib()

    def call(x=fake((2, 3, 10, 16)), pos=fake((10, 2), torch.int64), axes=(8, 8), theta=1e4, y=fake((2, 3, 10, 16))):
        dims = (C.c_int32 * max(1, len(axes)))(*axes)
        return lib.llsa_rope_axes(ref(x) if x is not None else None, ref(pos) if pos is not None else None, len(axes), dims, theta, 0, ref(y) if y is not None else None,
                                  None)

    assert call(x=None) == ERR_NULL and call(pos=None) == ERR_NULL and call(y=None) == ERR_NULL
    assert call(x=fake((2, 3, 10, 16), torch.int32)) == ERR_DTYPE and call(y=fake((2, 3, 10, 16), F32)) == ERR_DTYPE and call(pos=fake((10, 2), BF16)) == ERR_DTYPE
    assert call(x=fake((3, 10, 16))) == ERR_SHAPE and call(y=fake((2, 3, 11, 16))) == ERR_SHAPE and call(pos=fake((9, 2), torch.int64)) == ERR_SHAPE
    assert call(pos=fake((10, 3), torch.int64)) == ERR_SHAPE and call(pos=fake((1, 10, 2), torch.int64)) == ERR_SHAPE and call(axes=(8, 6)) == ERR_SHAPE
    assert call(x=fake((1, 1, 1, 514)), y=fake((1, 1, 1, 514)), pos=fake((1, 1), torch.int64), axes=(514,)) == ERR_SHAPE
    assert call(axes=()) == ERR_ARG and call(axes=(4, 4, 4, 2, 2)) == ERR_ARG and call(axes=(9, 7)) == ERR_ARG and call(axes=(16, 0)) == ERR_ARG
    for theta in (0.0, -1.0, float("inf"), float("nan")):
        assert call(theta=theta) == ERR_ARG
    assert call(x=fake((2, 3, 10, 16), strides=(960, 320, 32, 2))) == ERR_STRIDE and call(pos=fake((10, 2), torch.int64, strides=(4, 2))) == ERR_STRIDE
    assert call(x=fake((2, 3, 0, 16)), y=fake((2, 3, 0, 16)), pos=fake((0, 2), torch.int64)) == OK


def test_operators_refuse_tensors_on_the_cpu():
    import llsa_b200
    x, w = torch.zeros(2, 4, 16), torch.zeros(8, 16)
    for call in (lambda: llsa_b200.layer_norm(x), lambda: llsa_b200.linear(x, w), lambda: llsa_b200.linear(x, w, activation="gelu_tanh"),
                 lambda: llsa_b200.rope_axes(torch.zeros(1, 2, 4, 16), torch.zeros(4, 1), (16,))):
        with pytest.raises(RuntimeError, match="CUDA|cuda"):
            call()
