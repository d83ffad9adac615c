"""Gradients of the cross-entropy of a linear layer where p does not fit at once, bf16: several pieces of the classes, a shorter last one among them, whose
parts of dx are added up. Against the formulas in 64 bits; tolerances as in test_gpu_train_ce.py, for which the rows of a sum over all of them count once.
"""
import ctypes as C

import pytest
import torch

from test_gpu_train_ce import BF16, E, IGNORED, U, formulas, inputs, near

pytestmark = pytest.mark.gpu


def workspace(x, w, t, forward):
    from mimir_b200 import _lib
    d, need = _lib.LinearCeDesc(), C.c_uint64()
    (d.n, d.d), d.v = x.shape, w.shape[1]
    d.x, d.w, d.targets = x.data_ptr(), w.data_ptr(), t.data_ptr()
    d.dtype, d.target_dtype, d.w_layout, d.has_ignore, d.ignore_index = _lib.BF16, _lib.I64, _lib.B_KN if w.is_contiguous() else _lib.B_NK, 1, IGNORED
    assert _lib.lib().mimk_linear_ce_workspace(C.byref(d), int(forward), 1, C.byref(need)) == 0
    return need.value


def in_parts(x, w, t, rows):
    """(losses, lse, dx) of each `rows` rows, then dw of all of them, of the sum of the losses, each with its bound."""
    parts, total, spread, terms = [], 0.0, 0.0, 0.0
    for i in range(0, x.shape[0], rows):
        want, kept = formulas(x[i:i + rows], w, t[i:i + rows], mean=False)
        parts.append((i, want))
        xi, ti = torch.where(kept[:, None], x[i:i + rows].double(), 0.0), torch.where(kept, t[i:i + rows], 0)[:, None]
        l = xi @ w.double()
        el = xi.abs() @ w.double().abs() * (x.shape[1] * E / 2)
        lse = torch.logsumexp(l, 1, keepdim=True)
        p = torch.exp(l - lse)
        dl = p.scatter_add(1, ti, -torch.ones_like(lse)) * kept[:, None]
        edl = p * ((el + (el.max(1, keepdim=True).values + 8 * E + E * lse.abs())) * 1.01 + E * (8 + (l - lse).abs()))
        edl = edl.scatter_add(1, ti, torch.full_like(lse, E)) * kept[:, None] + (4 * E + U) * dl.abs()
        total, spread, terms = total + xi.t() @ dl, spread + xi.t().abs() @ edl, terms + xi.t().abs() @ dl.abs()
    return parts, (total, 1.02 * (spread + x.shape[0] * E * terms + U * total.abs()) + 1e-37)


# pieces of 4096, 4096 and 108 classes; three of 32768 and one more, then 50: k-blocks of dx dealt out over two tiles, of which the last piece has
# one, and more than 2^30 logits, whose exponentials are not kept
@pytest.mark.parametrize("shape,rows", [((70000, 16, 8300), 5000), ((8192, 64, 4 * 32768 + 50), 1024)])
@pytest.mark.parametrize("masked", [0.0, 0.2])
@pytest.mark.parametrize("nk", [False, True])
def test_gradients_by_pieces(shape, rows, masked, nk):
    from mimir_b200 import tensor as T
    x, w, t = inputs(*shape, BF16, nk, masked=masked)
    ignore = IGNORED if masked else None
    parts, dw_want = in_parts(x, w, t, rows)
    lse = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="none", return_lse=True)[1]
    calls = {"from lse": (False, lambda: T.linear_cross_entropy_grad(x, w, t, lse, ignore_index=ignore, reduction="sum"))}
    if shape[0] * shape[2] > 2 ** 30:
        calls["at once"] = (True, lambda: T.linear_cross_entropy_with_grad(x, w, t, ignore_index=ignore, reduction="sum")[1:])
    for name, (forward, call) in calls.items():
        assert workspace(x, w, t, forward) < 2 * shape[0] * shape[2], "p is in one piece"
        dx, dw = call()
        again = call()
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]), name
        for i, want in parts:
            assert near(lse[i:i + rows], *want[1]) and near(dx[i:i + rows], *want[2]), (name, i)
        assert near(dw, *dw_want), name
    T.device_status()
