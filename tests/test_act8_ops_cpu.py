"""What the 8-bit training operators refuse without a GPU: CPU tensors, and at the C ABI every size, pitch and pointer that a kernel
does not take (all checked before anything is launched)."""
import ctypes as C

import pytest
import torch

from act8_ref import held8
from hcmoco_amd import _lib, hip_ops

Z, P = C.c_void_p(0), C.c_void_p(4096)      # P: never read, the call ends at its checks


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(8)
    for call in (lambda: hip_ops.act8_pack(x), lambda: hip_ops.layer_norm(x), lambda: hip_ops.layer_norm(x, w, w, act8=True),
                 lambda: hip_ops.fp8_weight(x), lambda: hip_ops.fp8_linear(x, x)):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()


def test_pitches():
    L = _lib.lib()
    for c, p, s in ((1, 16, 4), (16, 16, 4), (17, 32, 4), (128, 128, 4), (512, 512, 4), (513, 528, 8), (1290, 1296, 12)):
        assert (L.hcm_act8_pitch(c), L.hcm_act8_scale_pitch(c)) == (p, s)


def test_pack_refuses():
    L = _lib.lib()
    good = dict(x=P, dt=0, rows=4, cols=270, ldx=270, q=P, ldq=272, s=P, lds=4)
    for bad in (dict(x=Z), dict(dt=3), dict(dt=-1), dict(rows=0), dict(rows=-1), dict(cols=0), dict(ldx=269), dict(q=Z), dict(q=C.c_void_p(4100)),
                dict(ldq=270), dict(ldq=288), dict(s=Z), dict(lds=3), dict(rows=2 ** 31)):
        a = {**good, **bad}
        assert L.hcm_act8_pack(a['x'], a['dt'], a['rows'], a['cols'], a['ldx'], a['q'], a['ldq'], a['s'], a['lds'], Z) != 0, bad
        if 'ldx' not in bad:
            assert L.hcm_act8_unpack(a['q'], a['ldq'], a['s'], a['lds'], a['rows'], a['cols'], a['x'], a['dt'], Z) != 0, bad


def test_weight_pack_refuses():
    L = _lib.lib()
    good = dict(w=P, dt=0, rows=200, cols=270, ldw=270, q=P, ldq=272, s=P, lds=4, qt=P, ldqt=208, st=P, ldst=4)
    for bad in (dict(w=Z), dict(dt=7), dict(rows=0), dict(cols=0), dict(ldw=1), dict(q=Z), dict(ldq=270), dict(s=Z), dict(lds=8), dict(qt=Z),
                dict(ldqt=200), dict(st=Z), dict(ldst=2), dict(qt=C.c_void_p(4104))):
        a = {**good, **bad}
        assert L.hcm_fp8_weight_pack(*[a[k] for k in good], Z) != 0, bad


def test_layer_norm_refuses():
    L = _lib.lib()
    good = dict(x=P, dt=0, rows=4, cols=270, ldx=270, w=Z, wd=0, b=Z, bd=0, eps=1e-5, y=P, mean=P, rstd=P, q=P, ldq=272, s=P, lds=4)
    for bad in (dict(x=Z), dict(dt=3), dict(rows=0), dict(rows=2 ** 31), dict(cols=0), dict(ldx=269), dict(wd=5), dict(bd=-2), dict(y=Z), dict(mean=Z),
                dict(s=Z), dict(q=C.c_void_p(4100)), dict(ldq=270), dict(lds=1)):
        a = {**good, **bad}
        assert L.hcm_layer_norm_forward(*[a[k] for k in good], Z) != 0, bad
    need = L.hcm_layer_norm_backward_workspace_bytes(4, 270)
    assert need > 0 and L.hcm_layer_norm_backward_workspace_bytes(0, 270) == 0
    good = dict(x=P, ldx=270, q=Z, ldq=0, s=Z, lds=0, dy=P, dt=0, rows=4, cols=270, w=Z, wd=0, mean=P, rstd=P, dx=P, dw=P, db=P, bd=0, ws=P, n=need)
    for bad in (dict(x=Z), dict(q=P), dict(q=P, s=P), dict(x=Z, q=P, s=P, ldq=270, lds=4), dict(dy=Z), dict(rows=0), dict(dx=Z), dict(mean=Z),
                dict(ws=Z), dict(n=need - 1), dict(dt=4), dict(ldx=3)):
        a = {**good, **bad}
        assert L.hcm_layer_norm_backward(*[a[k] for k in good], Z) != 0, bad


def test_products_refuse():
    L = _lib.lib()
    good = dict(x=P, ldx=272, sx=P, ldsx=4, w=P, ldw=272, sw=P, ldsw=4, b=Z, bd=0, M=4, N=200, K=270, y=P, od=0, ws=P, n=1 << 30)
    for bad in (dict(x=Z), dict(ldx=270), dict(sx=Z), dict(ldsx=3), dict(w=Z), dict(ldw=288), dict(sw=Z), dict(ldsw=8), dict(b=P, bd=3), dict(M=0),
                dict(M=2 ** 31 - 1), dict(N=0), dict(N=2 ** 22 + 1), dict(K=0), dict(K=2 ** 22 + 1), dict(y=Z), dict(od=-1), dict(od=3),
                dict(x=C.c_void_p(4104)), dict(w=C.c_void_p(4104)), dict(sx=C.c_void_p(4097)), dict(sw=C.c_void_p(4098))):
        a = {**good, **bad}
        assert L.hcm_fp8_matmul(*[a[k] for k in good], Z) != 0, bad
    need = L.hcm_fp8_matmul_workspace_bytes(64, 128, 4096)
    assert need > 0 and L.hcm_fp8_matmul_workspace_bytes(8192, 8192, 8192) == 0 and L.hcm_fp8_matmul_workspace_bytes(0, 1, 1) == 0
    a = {**good, **dict(ldx=4096, ldw=4096, ldsx=32, ldsw=32, M=64, N=128, K=4096)}
    for bad in (dict(n=need - 1), dict(ws=Z)):
        assert L.hcm_fp8_matmul(*[{**a, **bad}[k] for k in good], Z) != 0, bad
    good = dict(x=P, dt=0, ldx=270, w=P, ldw=272, sw=P, ldsw=4, b=Z, bd=0, M=4, N=200, K=270, y=P, q=Z, s=Z)
    for bad in (dict(x=Z), dict(dt=3), dict(ldx=269), dict(w=Z), dict(ldw=270), dict(sw=Z), dict(ldsw=3), dict(b=P, bd=4), dict(M=0), dict(M=33),
                dict(N=0), dict(K=0), dict(y=Z), dict(q=P), dict(s=P), dict(w=C.c_void_p(4100)), dict(q=C.c_void_p(4100), s=P),
                dict(M=9, K=3712, ldx=3712, ldw=3712, ldsw=32)):
        a = {**good, **bad}
        assert L.hcm_fp8_rows(*[a[k] for k in good], Z) != 0, bad
    assert [L.hcm_fp8_rows_supported(*a) for a in ((1, 32768), (1, 32769), (32, 1024), (32, 1025), (33, 1), (0, 1))] == [1, 0, 1, 0, 0, 0]
    need = L.hcm_fp8_wgrad_workspace_bytes(4000, 200, 270, 0, 1)
    assert need > 0 and L.hcm_fp8_wgrad_workspace_bytes(8192, 4096, 4096, 1, 1) == 0
    good = dict(x=P, ldx=272, sx=P, ldsx=4, dy=P, dd=0, M=4000, N=200, K=270, dw=P, wd=0, db=P, bd=0, ws=P, n=need)
    for bad in (dict(x=Z), dict(ldx=270), dict(sx=Z), dict(ldsx=2), dict(dy=Z), dict(dd=3), dict(M=0), dict(M=2 ** 31), dict(N=0), dict(K=0),
                dict(N=2 ** 22 + 1), dict(dw=Z, db=Z), dict(wd=9), dict(bd=-1), dict(ws=Z), dict(n=need - 1), dict(x=C.c_void_p(4104)), dict(dy=C.c_void_p(4104))):
        a = {**good, **bad}
        assert L.hcm_fp8_wgrad(*[a[k] for k in good], Z) != 0, bad


def test_sizes_past_a_launch_are_refused():
    L, bad = _lib.lib(), 1      # hipErrorInvalidValue, not a launch that the runtime turned down
    assert L.hcm_act8_pack(P, 0, 2 ** 30, 1, 1, P, 16, P, 4, Z) == bad
    assert L.hcm_act8_unpack(P, 16, P, 4, 2 ** 30, 1, P, 0, Z) == bad
    for rows, cols in ((1, 2 ** 27), (2 ** 22, 16385)):
        assert L.hcm_layer_norm_forward(P, 0, rows, cols, cols, Z, 0, Z, 0, 1e-5, P, P, P, Z, 0, Z, 0, Z) == bad
        n = L.hcm_layer_norm_backward_workspace_bytes(rows, cols)
        assert L.hcm_layer_norm_backward(P, cols, Z, 0, Z, 0, P, 0, rows, cols, Z, 0, P, P, P, P, P, 0, P, n, Z) == bad
    M, N, K = 2 ** 31 - 1000, 2 ** 22, 128
    assert L.hcm_fp8_matmul(P, 128, P, 4, P, 128, P, 4, Z, 0, M, N, K, P, 1, P, 1 << 60, Z) == bad


def test_the_format_of_the_reference_matches_torchs_e4m3():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 300, generator=g) * torch.exp(4 * torch.randn(50, 1, generator=g))
    val, e = held8(x)
    s = torch.repeat_interleave(torch.exp2(e.double()), 128, 1)[:, :300]
    assert torch.equal((x.double() / s).float().to(torch.float8_e4m3fn).double() * s, val)
    assert (x.double() / s).abs().max() <= 448
    blocks = torch.nn.functional.pad((x.double() / s).abs(), (0, 84)).view(50, 3, 128).amax(2)
    assert (blocks > 224).all()                            # a smaller power of two would not have held the block


def test_the_bounds_that_act8_pack_states():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(400, 256, generator=g) * torch.exp(4 * torch.randn(400, 256, generator=g))
    x[0, :2] = torch.tensor([225., 7.5 * 2.0 ** -9])          # within 2^14 of the largest, and off by more than 2^-4 of itself
    val, e = held8(x)
    scale = torch.repeat_interleave(torch.exp2(e.double()), 128, 1)
    off, mag = (val - x.double()).abs(), x.double().abs()
    assert (off <= torch.maximum(mag / 16, scale / 1024)).all()
    top = torch.repeat_interleave(mag.view(400, 2, 128).amax(2), 128, 1)
    assert (off <= mag / 16)[mag * 8192 >= top].all() and off[0, 1] > mag[0, 1] / 16
    L = _lib.lib()
    per = lambda c: (L.hcm_act8_pitch(c) + L.hcm_act8_scale_pitch(c)) / c
    assert (per(8), per(16)) == (2.5, 1.25) and per(4096) < 1.01
