"""CPU: the C entries of cross attention, RMS norm and gradient clipping refuse what their kernels do not take before anything is launched (the addresses below are
never read), and the Python entries refuse tensors that are not on a GPU."""
import ctypes
import math

import pytest
import torch

from ogmm_amd import _lib, ops, train_ops
from ogmm_amd._lib import OgmmError


@pytest.fixture(scope="module")
def lib():
    import os
    import __graft_entry__ as g
    if not os.path.isfile(_lib.LIB_PATH):
        g.build()
    return _lib.load()


def xattn(**kw):
    a = _lib.XattnDesc()
    a.q = a.k = a.v = a.o = a.lse = a.dout = a.dq = a.dk = a.dv = a.workspace = 4096
    a.B, a.Nq, a.Nk, a.H, a.Hkv, a.d, a.type, a.scale = 2, 16, 32, 4, 2, 64, 1, 0.125
    a.q_b, a.q_n, a.q_h = a.do_b, a.do_n, a.do_h = 16 * 256, 256, 64
    a.k_b, a.k_n, a.k_h = a.v_b, a.v_n, a.v_h = 32 * 128, 128, 64
    for name, value in kw.items():
        setattr(a, name, value)
    return a


BAD_ATTENTION = [dict(B=-1), dict(Nq=-1), dict(Nk=-5), dict(H=0), dict(Hkv=0), dict(H=3), dict(d=0), dict(d=4), dict(d=60), dict(d=136), dict(type=3), dict(type=-1),
                 dict(q_n=255), dict(k_h=65), dict(v_b=4), dict(q=4098), dict(k=4104), dict(v=4097), dict(o=4104), dict(q=None), dict(k=None), dict(v=None), dict(o=None),
                 dict(k_n=1 << 24), dict(q_h=1 << 24), dict(q_n=-256), dict(scale=math.nan), dict(scale=math.inf), dict(B=1 << 20, H=1 << 16, Hkv=1, Nq=1 << 20),
                 dict(B=1 << 24, H=1, Hkv=1, Nq=1, Nk=1, d=8), dict(B=1, H=1, Hkv=1, Nq=1, Nk=(1 << 30) + 1), dict(B=1 << 30, H=1 << 30, Hkv=1 << 30)]


@pytest.mark.parametrize("kw", BAD_ATTENTION, ids=str)
def test_attention_forward_refuses(lib, kw):
    assert lib.ogmm_xattn_fwd(ctypes.byref(xattn(**kw)), None) != 0
    assert b"ogmm_xattn_fwd" in lib.ogmm_last_error()


@pytest.mark.parametrize("kw", BAD_ATTENTION + [dict(dout=None), dict(lse=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(do_n=100), dict(dq=4104), dict(dout=4100)], ids=str)
def test_attention_backward_refuses(lib, kw):
    assert lib.ogmm_xattn_bwd(ctypes.byref(xattn(**kw)), None) != 0
    assert b"ogmm_xattn_bwd" in lib.ogmm_last_error()


def test_attention_of_nothing_and_the_struct(lib):
    assert lib.ogmm_xattn_fwd(None, None) != 0 and lib.ogmm_xattn_bwd(None, None) != 0
    assert lib.ogmm_xattn_fwd(ctypes.byref(xattn(B=0)), None) == 0 and lib.ogmm_xattn_bwd(ctypes.byref(xattn(B=0)), None) == 0
    assert lib.ogmm_xattn_workspace_bytes(ctypes.byref(xattn()), 0) >= 0 and lib.ogmm_xattn_workspace_bytes(ctypes.byref(xattn()), 1) >= 0


def test_struct_matches_the_header():
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ogmm_hip.h")).read()
    body = header[header.index("typedef struct ogmm_xattn {"):header.index("} ogmm_xattn;")]
    fields = re.findall(r"[\*\s]([A-Za-z_0-9]+)\s*[;,]", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
    assert fields == [f[0] for f in _lib.XattnDesc._fields_]
    assert ops._XATTN.size == ctypes.sizeof(_lib.XattnDesc)
    values = list(range(1, 36))
    got = _lib.XattnDesc.from_buffer_copy(ops._XATTN.pack(*values))
    assert [getattr(got, f) for f in fields] == values


def norm_args(**kw):
    a = dict(x=4096, ldx=64, r=None, ldr=0, w=4096, rows=10, D=64, type=1, wtype=0, eps=1e-6)
    a.update(kw)
    return [a[n] for n in ("x", "ldx", "r", "ldr", "w", "rows", "D", "type", "wtype", "eps")]


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(D=0), dict(D=32769), dict(type=5), dict(wtype=2), dict(type=0, wtype=1), dict(w=None), dict(x=None), dict(eps=-1.0), dict(eps=math.nan)], ids=str)
def test_norm_refuses(lib, kw):
    assert lib.ogmm_rms_norm(*norm_args(**kw), 4096, None, None, None) != 0
    assert lib.ogmm_rms_norm_q8(*norm_args(**kw), 0, 4096, 4096, None, None) != 0
    a = norm_args(**kw)
    if "eps" not in kw and "x" not in kw:
        assert lib.ogmm_rms_norm_bwd(4096, 64, 4096, 64, None, 0, a[4], 4096, None, 0, a[5], a[6], a[7], a[8], 4096, 4096, 4096, None) != 0


def test_norm_refuses_missing_outputs_and_groups(lib):
    assert lib.ogmm_rms_norm(*norm_args(), None, None, None, None) != 0
    assert lib.ogmm_rms_norm(*norm_args(r=4096), 4096, None, None, None) != 0          # a residual without a place for the sum
    for group in (-32, 1, 16, 96, 256):
        assert lib.ogmm_rms_norm_q8(*norm_args(), group, 4096, 4096, None, None) != 0
    assert lib.ogmm_rms_norm_q8(*norm_args(), 0, 4096, None, None, None) != 0
    assert lib.ogmm_rms_norm(*norm_args(rows=0, x=None), None, None, None, None) == 0
    assert lib.ogmm_rms_norm_bwd(4096, 64, 4096, 64, 4096, 64, 4096, 4096, None, 0, 10, 64, 0, 0, 4096, 4096, 4096, None) != 0          # fp32 rows as two summands
    assert lib.ogmm_rms_norm_bwd_workspace_bytes(-1, 8) == -1 and lib.ogmm_rms_norm_bwd_workspace_bytes(10, 8) >= 10 * 8 * 4


def lists(ptrs, numel, types):
    n = len(ptrs)
    return n, (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numel), (ctypes.c_int32 * n)(*types)


def test_clipping_refuses(lib):
    good = lists([4096, 8192], [10, 20], [0, 1])
    tail = (1.0, 1.0, 4096, 4096, None)          # inv_scale, max_norm, norm, workspace, stream
    bad = [
        (lists([4096, 4096], [10, 20], [0, 0]), None, tail), (lists([4096, 4100], [2, 20], [0, 0]), None, tail), (lists([8192, 4096], [10, 2049], [1, 1]), None, tail),
        (lists([4096], [10], [3]), None, tail), (lists([4096], [-1], [0]), None, tail), (lists([None], [4], [0]), None, tail), (lists([4098], [4], [0]), None, tail),
        (lists([4097], [4], [1]), None, tail), (good, None, (0.0, 1.0, 4096, 4096, None)), (good, None, (math.nan, 1.0, 4096, 4096, None)),
        (good, None, (1.0, -1.0, 4096, 4096, None)), (good, None, (1.0, math.nan, 4096, 4096, None)), (good, None, (1.0, 1.0, None, 4096, None)), (good, None, (1.0, 1.0, 4096, None, None)),
        (good, [16384, 16400], tail), (good, [8192, 16384], tail), (good, [16384, 8192], tail), (good, [16384, 16426], tail), (good, [16384, None], tail)]
    for i, ((n, p, c, t), out, rest) in enumerate(bad):
        o = None if out is None else (ctypes.c_void_p * n)(*out)
        assert lib.ogmm_clip_grads(n, p, c, t, o, *rest) != 0, i
        assert b"ogmm_clip_grads" in lib.ogmm_last_error()
    n, p, c, t = lists([4096], [4], [7])
    assert lib.ogmm_grad_norm(n, p, c, t, 1.0, 4096, 4096, None) != 0
    assert lib.ogmm_grad_norm(-1, None, None, None, 1.0, 4096, 4096, None) != 0
    assert lib.ogmm_grad_norm_workspace_bytes(-1, None) == -1
    _, _, c, _ = lists([0] * 1000, [5] * 999 + [1 << 33], [0] * 1000)
    assert lib.ogmm_grad_norm_workspace_bytes(1000, c) == 5 * 512 * 8          # 1007 pieces of at most 2^30 values, 230 to a launch


def test_tensors_on_the_cpu_are_refused():
    q, k = torch.ones(1, 4, 2, 8), torch.ones(1, 6, 2, 8)
    x, w = torch.ones(3, 8), torch.ones(8)
    for f in (lambda: ops.cross_attention(q, k, k), lambda: train_ops.cross_attention(q, k, k), lambda: ops.rms_norm(x, w), lambda: train_ops.rms_norm(x, w, x),
              lambda: ops.rms_norm_q8(x, w), lambda: ops.rms_norm_bwd(x, x, w, torch.ones(3)), lambda: ops.grad_norm([x]), lambda: ops.clip_grads_([x], 1.0), lambda: ops.grad_norm([None])):
        with pytest.raises(OgmmError):
            f()


def test_a_workspace_that_is_not_aligned_is_refused(lib):
    a = xattn(B=1, Nq=1, Nk=4096)          # few rows, many keys: cut into parts
    assert lib.ogmm_xattn_workspace_bytes(ctypes.byref(a), 0) > 0
    for ws in (None, 4104):
        a.workspace = ws
        assert lib.ogmm_xattn_fwd(ctypes.byref(a), None) != 0 and lib.ogmm_xattn_bwd(ctypes.byref(a), None) != 0


def test_which_tensors_are_without_gaps():
    x = torch.zeros(4, 6, 5)
    for t in (x, x.permute(2, 0, 1), x[1:], x[:, :, :0], x[:0], torch.zeros(3, 0), torch.zeros(0, 3), torch.zeros(()), x[:, :1, :1][:1], torch.zeros(2, 3, 4, 5).contiguous(memory_format=torch.channels_last)):
        assert ops._dense(t), (t.shape, t.stride())
    for t in (x[:, 1:], x[:, :, ::2], torch.zeros(1, 5).expand(4, 5), x.as_strided((4, 4), (1, 1))):
        assert not ops._dense(t), (t.shape, t.stride())


def test_trainer_refuses_a_negative_limit():
    from ogmm_amd.trainer import Trainer
    model = torch.nn.Linear(2, 2)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            Trainer(model, max_grad_norm=bad)
    assert Trainer(model).max_grad_norm is None
