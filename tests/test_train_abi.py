"""Arguments that the training operators' C entry points refuse before they look for a device."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry
    entry.build()
    from mimir_b200 import _lib
    return _lib


def test_gated_mlp(lib):
    L = lib.lib()
    for fn in (L.mimk_mlp_gated_fwd, L.mimk_mlp_gated_bwd):
        assert fn(None, None) == 1
        d = lib.MlpTrainDesc()
        d.m, d.k, d.f, d.n, d.dtype = 4, 8, 8, -8, lib.BF16
        assert fn(C.byref(d), None) == 1
        d.n, d.dtype = 8, lib.F32
        assert fn(C.byref(d), None) == 4
        d.dtype, d.b_layout = lib.BF16, 2
        assert fn(C.byref(d), None) == 1
        d.b_layout, d.f = lib.B_NK, 1 << 30
        assert fn(C.byref(d), None) == 8
    assert L.mimk_mlp_gated_train_sizes(None, None, None, None) == 1


def test_linear_cross_entropy(lib):
    L = lib.lib()
    need = C.c_uint64()
    for fn in (L.mimk_linear_ce_fwd, L.mimk_linear_ce_bwd, L.mimk_linear_ce_fwd_bwd):
        assert fn(None, None) == 1
        d = lib.LinearCeDesc()
        d.n, d.d, d.v, d.dtype, d.target_dtype = -1, 8, 8, lib.BF16, lib.I64
        assert fn(C.byref(d), None) == 1
        d.n, d.dtype = 4, lib.I32
        assert fn(C.byref(d), None) == 4
        d.dtype, d.target_dtype = lib.F32, lib.F32
        assert fn(C.byref(d), None) == 4
        d.target_dtype, d.reduction = lib.I32, 3
        assert fn(C.byref(d), None) == 1
        d.reduction, d.w_layout = lib.REDUCTION_SUM, -1
        assert fn(C.byref(d), None) == 1
        d.w_layout, d.v = lib.B_KN, 1 << 30
        assert fn(C.byref(d), None) == 8
        d.v = 0
        assert fn(C.byref(d), None) == 2                     # rows, and no class
    assert L.mimk_linear_ce_workspace(None, 1, 1, C.byref(need)) == 1


def test_norm_and_clipping(lib):
    L = lib.lib()
    p, n, dt = (C.c_void_p * 1)(16), (C.c_int64 * 1)(-1), (C.c_int32 * 1)(lib.F32)
    assert L.mimk_grad_norm(p, n, dt, -1, 16, 16, 1 << 20, None) == 1
    assert L.mimk_grad_norm(p, n, dt, 1, 16, 16, 1 << 20, None) == 1         # a negative length
    n[0] = 8
    assert L.mimk_grad_norm(None, n, dt, 1, 16, 16, 1 << 20, None) == 1
    assert L.mimk_grad_norm(p, n, dt, 1, None, 16, 1 << 20, None) == 1       # nowhere to put the norm
    dt[0] = lib.I32
    assert L.mimk_grad_norm(p, n, dt, 1, 16, 16, 1 << 20, None) == 4
    dt[0], p[0] = lib.F32, 18
    assert L.mimk_grad_norm(p, n, dt, 1, 16, 16, 1 << 20, None) == 3
    p[0] = None
    assert L.mimk_grad_norm(p, n, dt, 1, 16, 16, 1 << 20, None) == 1
    p[0] = 16
    assert L.mimk_clip_grads(p, None, n, dt, 1, 1.0, 0.0, 16, 16, 1 << 20, None) == 1
    assert L.mimk_clip_grads(p, p, n, dt, 1, -1.0, 0.0, 16, 16, 1 << 20, None) == 1
    assert L.mimk_clip_grads_workspace(-1, C.byref(C.c_uint64())) == 1
