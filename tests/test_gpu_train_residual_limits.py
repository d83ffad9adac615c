"""The step between blocks at the ends of what its descriptor may hold."""
import ctypes as C

import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def call(p, dr, dx, gate_rows):
    """Both passes by the C entry points: (r_out, x, dr, dh, dgamma, dpost_gamma, dgate)."""
    from mimir_b200 import _lib as L
    n, features = p["r"].shape
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    code = lambda t: L.BF16 if t.dtype == BF16 else L.F32  # noqa: E731
    new = lambda t: None if t is None else torch.full_like(t, float("nan"))  # noqa: E731
    out = [new(p["r"]), new(p["h"]), new(p["r"]), new(p["h"]), new(p["gamma"]), new(p["post_gamma"]), new(p["gate"])]
    kept = torch.empty((2, n), device="cuda")
    d = L.ResidualRmsnormDesc()
    d.n, d.d, d.gate_rows, d.eps, d.residual_scale, d.branch_scale = n, features, gate_rows, 1e-6, 1.0, 1.0
    d.r, d.h, d.gamma, d.post_gamma, d.gate = (at(p[k]) for k in ("r", "h", "gamma", "post_gamma", "gate"))
    d.stream_dtype, d.block_dtype, d.gamma_dtype, d.gate_dtype = code(p["r"]), code(p["h"]), code(p["gamma"]), code(p["gate"])
    if p["post_gamma"] is not None:
        d.post_gamma_dtype = code(p["post_gamma"])
    d.r_out, d.x, d.kept = at(out[0]), at(out[1]), at(kept)
    stream, lib, need = torch.cuda.current_stream().cuda_stream, L.lib(), C.c_uint64()
    assert lib.mimk_residual_rmsnorm_fwd(C.byref(d), stream) == 0
    d.dr_out, d.dx = at(dr), at(dx)
    d.dr, d.dh, d.dgamma, d.dpost_gamma, d.dgate = (at(t) for t in out[2:])
    assert lib.mimk_residual_rmsnorm_workspace(C.byref(d), C.byref(need)) == 0
    room = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = room.data_ptr(), need.value
    assert lib.mimk_residual_rmsnorm_bwd(C.byref(d), stream) == 0
    return out


def off16(t):
    """The same values, not on 16 bytes."""
    return torch.cat([t.new_empty(1), t.reshape(-1)])[1:].view(t.shape)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("shape", [(50, 256), (50, 257), (9, 8192), (5, 12000)])
def test_one_gate_row_for_any_number_of_rows(shape, post):
    """gate_rows may be more than there are rows, up to the largest number: the gate's one row is for all of them."""
    n, features = shape
    for stream, block in ((BF16, BF16), (F32, BF16), (F32, F32)):
        p = dict(r=randn(shape, 1, 2.0, stream), h=randn(shape, 2, 0.7, block), gamma=randn((features,), 3, 1.0, stream), gate=randn((1, features), 4, 1.0, block),
                 post_gamma=randn((features,), 5, 1.0, stream) if post else None)
        dr, dx = randn(shape, 6, 1.0, stream), randn(shape, 7, 1.0, block)
        for shift in (lambda t: t, off16):
            q = {k: None if t is None else shift(t) for k, t in p.items()}
            want = call(q, shift(dr), shift(dx), n)
            assert not any(bool(t.isnan().any()) for t in want if t is not None)
            for rows in (n + 1, 1 << 31, 2 ** 63 - n, 2 ** 63 - 1):
                got = call(q, shift(dr), shift(dx), rows)
                assert all((g is None and w is None) or torch.equal(g, w) for g, w in zip(got, want)), (rows, stream, block)
