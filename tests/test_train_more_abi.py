"""Arguments that the C entry points of the embedding, the norms between blocks and the orthogonalised update refuse before they look for a device."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry
    entry.build()
    from mimir_b200 import _lib
    return _lib


def test_embedding(lib):
    L, need = lib.lib(), C.c_uint64()
    for fn in (L.mimk_embedding, L.mimk_embedding_grad):
        assert fn(None, None) == 1
        d = lib.EmbeddingDesc()
        d.n, d.d, d.v, d.dtype, d.out_dtype, d.id_dtype = -1, 8, 8, lib.BF16, lib.BF16, lib.I64
        assert fn(C.byref(d), None) == 1
        d.n, d.dtype = 4, lib.I32
        assert fn(C.byref(d), None) == 4
        d.dtype, d.out_dtype = lib.BF16, lib.I64
        assert fn(C.byref(d), None) == 4
        d.out_dtype, d.id_dtype = lib.F32, lib.F32
        assert fn(C.byref(d), None) == 4
        d.id_dtype, d.v = lib.I32, 1 << 31
        assert fn(C.byref(d), None) == 8
    assert L.mimk_embedding_grad_workspace(None, C.byref(need)) == 1
    d.v = 100
    assert L.mimk_embedding_grad_workspace(C.byref(d), None) == 1


def test_residual_rmsnorm(lib):
    L, need = lib.lib(), C.c_uint64()

    def desc(**more):
        d = lib.ResidualRmsnormDesc()
        d.n, d.d, d.gate_rows, d.r, d.h, d.gamma, d.r_out, d.x, d.eps, d.residual_scale, d.branch_scale = 4, 8, 1, 256, 256, 256, 256, 256, 1e-6, 1.0, 1.0
        for k, v in more.items():
            setattr(d, k, v)
        return d
    for fn in (L.mimk_residual_rmsnorm_fwd, L.mimk_residual_rmsnorm_bwd):
        assert fn(None, None) == 1
        for status, more in ((1, dict(n=-1)), (1, dict(d=-1)), (1, dict(gate=256, gate_rows=0)), (1, dict(eps=-1.0)), (1, dict(eps=float("nan"))),
                             (4, dict(stream_dtype=lib.I32)), (4, dict(block_dtype=lib.I64)), (4, dict(stream_dtype=lib.BF16, block_dtype=lib.F32)),
                             (4, dict(gamma_dtype=lib.I32)), (4, dict(post_gamma=256, post_gamma_dtype=lib.I32)), (4, dict(gate=256, gate_dtype=lib.I64)),
                             (1, dict(h=None, post_gamma=256)), (1, dict(h=None, gate=256)), (1, dict(h=None, residual_scale=0.5)), (1, dict(h=None, gamma=None)),
                             (8, dict(d=32769)), (8, dict(n=1 << 31))):
            assert fn(C.byref(desc(**more)), None) == status, more
    assert L.mimk_residual_rmsnorm_workspace(None, C.byref(need)) == 1


def test_orthogonalize(lib):
    L, need = lib.lib(), C.c_uint64()
    x, c = (C.c_void_p * 1)(256), (C.c_float * 3)(1.5, -0.5, 0.0)

    def desc(**more):
        d = lib.OrthogonalizeDesc()
        d.batch, d.m, d.n, d.x, d.out, d.coefficients, d.eps, d.scale, d.steps, d.dtype = 1, 8, 8, x, 256, c, 1e-7, 1.0, 1, lib.F32
        for k, v in more.items():
            setattr(d, k, v)
        return d
    assert L.mimk_orthogonalize(None, None) == 1
    for status, more in ((1, dict(batch=-1)), (1, dict(m=-1)), (1, dict(n=-1)), (1, dict(steps=0)), (1, dict(eps=-1.0)), (1, dict(eps=float("nan"))), (4, dict(dtype=lib.I32)),
                         (8, dict(steps=65)), (8, dict(m=1 << 24))):
        assert L.mimk_orthogonalize(C.byref(desc(**more)), None) == status, more
        assert L.mimk_orthogonalize_workspace(C.byref(desc(**more)), C.byref(need)) == status, more
    # singular values that grow without limit: 6 s, and a step that takes 1 to 4.5
    for bad in ((6.0, 0.0, 0.0), (1.5, 1.5, 1.5), (float("nan"), 0.0, 0.0), (float("inf"), 0.0, 0.0)):
        assert L.mimk_orthogonalize(C.byref(desc(coefficients=(C.c_float * 3)(*bad))), None) == 8, bad
    assert L.mimk_orthogonalize_workspace(C.byref(desc(m=200, n=300)), C.byref(need)) == 0 and need.value >= 8 * 200 * 300
    assert L.mimk_orthogonalize_workspace(C.byref(desc()), C.byref(need)) == 0      # (small matrices take none)
    assert L.mimk_orthogonalize_workspace(C.byref(desc()), None) == 1
    # a stack of any length takes a bounded buffer
    many = (C.c_void_p * 4096)(*[256] * 4096)
    assert L.mimk_orthogonalize_workspace(C.byref(desc(batch=4096, m=1024, n=1024, x=many)), C.byref(need)) == 0 and need.value < 3 << 29


def test_as_many_rows_as_places_in_32_bits(lib):
    """Rows are numbered in 32 bits, with some to spare for the steps from one to the next."""
    L, need = lib.lib(), C.c_uint64()
    most = (1 << 31) - (1 << 17)
    d = lib.EmbeddingDesc()
    d.n, d.d, d.v, d.dtype, d.out_dtype, d.id_dtype = most, 1, 8, lib.BF16, lib.BF16, lib.I64
    assert L.mimk_embedding(C.byref(d), None) == L.mimk_embedding_grad(C.byref(d), None) == L.mimk_embedding_grad_workspace(C.byref(d), C.byref(need)) == 8
    d.n = most - 1
    assert L.mimk_embedding_grad_workspace(C.byref(d), C.byref(need)) == 0 and need.value >= 16 * most
    r = lib.ResidualRmsnormDesc()
    r.n, r.d, r.gate_rows, r.r, r.gamma, r.x, r.eps, r.residual_scale, r.branch_scale = most, 1, 1, 256, 256, 256, 1e-6, 1.0, 1.0
    assert L.mimk_residual_rmsnorm_fwd(C.byref(r), None) == L.mimk_residual_rmsnorm_bwd(C.byref(r), None) == L.mimk_residual_rmsnorm_workspace(C.byref(r), C.byref(need)) == 8
