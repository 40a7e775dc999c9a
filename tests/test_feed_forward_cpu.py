"""What the feed-forward operators refuse, without a GPU: CPU tensors at the Python entry points, and
bad shapes, types, strides, alignments and workspaces at the C entries, which return before any launch."""
import ctypes

import pytest
import torch

from graphsage_amd import _lib, functional, ops
from graphsage_amd.layers import GatedFeedForward
from graphsage_amd.models import GraphSAGE

P = ctypes.c_void_p(4096)          # never dereferenced: every call below is refused on the host
ODD = ctypes.c_void_p(4098)
EINVAL, EWORKSPACE, ELIMIT = -1, -2, -4


def test_cpu_tensors_are_refused():
    x, w, q, s = torch.zeros(3, 16), torch.ones(16), torch.zeros(3, 16, dtype=torch.int8), torch.ones(3)
    calls = [lambda: ops.rms_norm_fwd(x, w), lambda: ops.rms_norm_int8(x, w), lambda: ops.quantize_rows(x),
             lambda: ops.rms_norm_bwd(x, x, w), lambda: ops.dequantize_rows(q, s), lambda: ops.int8_linear(q, s, q, s),
             lambda: ops.int8_gated_linear(q, s, q, s, q, s), lambda: ops.gated_linear_fwd(x, x, x),
             lambda: ops.gated_linear_bwd(x, x, x, x, x), lambda: functional.rms_norm(x, w),
             lambda: functional.gated_linear(x, x, x), lambda: GatedFeedForward(16, 8)(x),
             lambda: GatedFeedForward(16, 8).quantize_()]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_layer_refuses_unknown_activations():
    with pytest.raises(RuntimeError, match="activation"):
        GatedFeedForward(8, 8, activation="tanh")
    with pytest.raises(RuntimeError, match="activation"):
        GraphSAGE(8, 8, ffn_channels=8, ffn_activation="swish")
    assert GraphSAGE(8, 8).blocks is None and len(GraphSAGE(8, 8, num_layers=4, ffn_channels=5).blocks) == 3


def refused(code, name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code, (name, args, _lib.last_error())
    assert name in _lib.last_error()


def norm(x=P, ldx=64, r=None, ldr=0, w=P, wd=0, rows=4, dim=64, dt=0, y=P, ldy=64, s=None, lds=0):
    return x, ldx, r, ldr, w, wd, rows, dim, dt, 1e-6, y, ldy, s, lds, None


@pytest.mark.parametrize("change", [dict(x=None), dict(w=None), dict(y=None), dict(dt=3), dict(wd=1), dict(dim=0), dict(rows=-1),
                                    dict(ldy=63), dict(s=P, lds=10), dict(ldx=-1)])
def test_rms_norm_fwd_refusals(change):
    refused(EINVAL, "sage_rms_norm_fwd", *norm(**change))


def test_norm_refusals():
    refused(ELIMIT, "sage_rms_norm_fwd", *norm(rows=1 << 31))
    ok = dict(x=P, ldx=64, r=None, ldr=0, w=None, wd=0, rows=4, dim=64, dt=0, eps=0.0, norm=0, q=P, ldq=64, cols=64, scale=P, s=None, lds=0, st=None)
    for change in (dict(q=None), dict(scale=None), dict(cols=63), dict(ldq=60), dict(dt=9), dict(cols=80)):
        refused(EINVAL, "sage_rms_norm_int8", *{**ok, **change}.values())
    ok = dict(q=P, ldq=8, scale=P, rows=2, dim=8, dt=1, out=P, ldo=8, st=None)
    for change in (dict(q=None), dict(out=None), dict(dt=7), dict(ldo=7), dict(dim=0)):
        refused(EINVAL, "sage_dequantize_rows", *{**ok, **change}.values())
    size = _lib.load().sage_rms_norm_bwd_workspace_bytes(100, 64, 0)
    assert size >= 64 * 4
    ok = dict(dy=P, ldy=64, s=P, lds=64, w=P, wd=0, ds=None, ldds=0, rows=100, dim=64, dt=0, eps=1e-6, dx=P, ldx=64, dw=P, ws=P, n=size, st=None)
    for code, change in ((EINVAL, dict(dy=None)), (EINVAL, dict(s=None)), (EINVAL, dict(w=None)), (EINVAL, dict(dx=None, dw=None)),
                         (EINVAL, dict(rows=0)), (EINVAL, dict(wd=2)), (EINVAL, dict(ldx=63)), (EWORKSPACE, dict(ws=None)), (EWORKSPACE, dict(n=size - 1))):
        refused(code, "sage_rms_norm_bwd", *{**ok, **change}.values())


def test_product_refusals():
    lib = _lib.load()
    size = lib.sage_product_workspace_bytes(512, 512, 8192, 0, 0)
    assert size > 0 and lib.sage_product_workspace_bytes(4, 512, 8192, 0, 0) == 0
    ok = dict(x=P, ldx=8192, xs=P, w=P, ldw=8192, ws=P, bias=None, m=512, n=512, k=8192, dt=0, out=P, ldo=512, wk=P, wn=size, st=None)
    for code, change in ((EINVAL, dict(x=None)), (EINVAL, dict(ws=None)), (EINVAL, dict(x=ODD)), (EINVAL, dict(ldw=8200)), (EINVAL, dict(k=8191)),
                         (EINVAL, dict(ldo=511)), (EINVAL, dict(dt=3)), (EINVAL, dict(n=0)), (ELIMIT, dict(k=131072)),
                         (ELIMIT, dict(ldx=1 << 23)), (EWORKSPACE, dict(wn=size - 1)), (EWORKSPACE, dict(wk=ODD))):
        refused(code, "sage_int8_linear", *{**ok, **change}.values())
    ok = dict(x=P, ldx=64, xs=P, g=P, ldg=64, gs=P, u=P, ldu=64, us=P, act=0, m=2, n=8, k=64, dt=0, out=P, ldo=8, wk=None, wn=0, st=None)
    for code, change in ((EINVAL, dict(u=None)), (EINVAL, dict(us=None)), (EINVAL, dict(act=3)), (EINVAL, dict(ldu=24, m=600)), (EINVAL, dict(k=24, m=600)), (EINVAL, dict(k=15)), (ELIMIT, dict(k=131072))):
        refused(code, "sage_int8_gated_linear", *{**ok, **change}.values())
    ok = dict(x=P, ldx=16, g=P, ldg=16, u=P, ldu=16, act=1, m=2, h=8, k=16, dt=1, out=P, ldo=8, saved=None, wk=None, wn=0, st=None)
    for change in (dict(x=None), dict(g=ODD, m=600), dict(act=-1), dict(dt=5), dict(k=12, m=600), dict(k=7), dict(ldx=20, m=600), dict(ldo=4), dict(h=0)):
        refused(EINVAL, "sage_gated_linear_fwd", *{**ok, **change}.values())
    size = lib.sage_gated_linear_bwd_workspace_bytes(20, 8, 16, 1)
    ok = dict(dh=P, ldh=8, x=P, ldx=16, g=P, ldg=16, u=P, ldu=16, saved=P, act=0, m=20, h=8, k=16, dt=1, dx=P, lddx=16, dw=P, ws=P, n=size, st=None)
    for code, change in ((EINVAL, dict(dh=None)), (EINVAL, dict(saved=None)), (EINVAL, dict(dx=None, dw=None)), (EINVAL, dict(m=0)), (EINVAL, dict(act=7)),
                         (EINVAL, dict(lddx=15)), (EWORKSPACE, dict(n=size - 1)), (EWORKSPACE, dict(ws=ODD))):
        refused(code, "sage_gated_linear_bwd", *{**ok, **change}.values())
    for change in (dict(i=None), dict(j=None), dict(l=None), dict(o=ODD), dict(ldo=24), dict(ldo=16), dict(b=0), dict(r=-1)):
        refused(EINVAL, "sage_pad_rows", *{**dict(i=P, ldi=20, r=3, j=P, ldj=20, rj=1, l=P, ldl=0, rl=2, b=20, o=P, ldo=32, st=None), **change}.values())


def test_empty_inputs_launch_nothing():
    lib = _lib.load()
    assert lib.sage_rms_norm_fwd(*norm(rows=0, x=None, y=None)) == 0
    assert lib.sage_int8_linear(None, 64, None, P, 64, P, None, 0, 8, 64, 0, None, 8, None, 0, None) == 0
    assert lib.sage_gated_linear_fwd(None, 16, P, 16, P, 16, 0, 0, 8, 16, 0, None, 8, None, None, 0, None) == 0
    assert lib.sage_pad_rows(None, 20, 0, None, 0, 0, None, 0, 0, 20, None, 32, None) == 0


def test_not_recordable_on_a_tape():
    with _lib.recording():
        with pytest.raises(RuntimeError, match="call tape"):
            ops._call("sage_pad_rows", torch.device("cuda", 0))
