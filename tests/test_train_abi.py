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
