"""The gated MLP block in training against its formulas in 64 bits, through the public operators.

Tolerances. u = 2^-8 is half the spacing of bf16 at 1. A result is rounded once (u |result|) and is a product one of whose operands (h, da
or db) was rounded before it (u times the product of the magnitudes). Sums of K terms in f32 add at most K 2^-23 times the product of the
magnitudes, through a, b and dh as well; exp and the division of the activation some units of 2^-22.
"""
import itertools

import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -22
BF16 = torch.bfloat16


def inputs(m, k, f, n, nk, seed=0, std=None):
    def weight(i, o, s):
        std_ = std or i ** -0.5
        return randn((o, i), s, std_, BF16).t() if nk else randn((i, o), s, std_, BF16)
    return (randn((m, k), seed, 1.0, BF16), weight(k, f, seed + 1), weight(k, f, seed + 2), weight(f, n, seed + 3), randn((m, n), seed + 4, 1.0, BF16))


def formulas(x, w1, w3, w2, dy):
    """(y, dx, dw1, dw3, dw2) and a bound of each one's error, in 64 bits."""
    x, w1, w3, w2, dy = (t.double() for t in (x, w1, w3, w2, dy))
    m, k, f, n = *x.shape, *w2.shape
    a, b, dh = x @ w1, x @ w3, dy @ w2.t()
    s = torch.sigmoid(a)
    g, ds = a * s, s + a * s * (1 - s)
    h, da, db = g * b, dh * b * ds, dh * g
    # errors of a, b, dh (f32 sums), and through the activation: |silu'| <= 1.1, |silu''| <= 0.5
    ea, eb, ed = k * E * (x.abs() @ w1.abs()), k * E * (x.abs() @ w3.abs()), n * E * (dy.abs() @ w2.t().abs())
    eg = 1.1 * ea + 8 * E * g.abs()
    eh = (eg * b.abs() + g.abs() * eb) * 1.01
    eda = (ed * (b * ds).abs() + dh.abs() * eb * 1.1 + (dh * b).abs() * (0.5 * ea + 16 * E)) * 1.01
    edb = (ed * g.abs() + dh.abs() * eg) * 1.01
    eh, eda, edb = eh + U * h.abs(), eda + U * da.abs(), edb + U * db.abs()

    def out(result, parts):
        bound = sum(p.abs() @ q.abs() * c + d for p, q, c, d in parts)
        return result, 1.02 * (U * result.abs() + bound) + 1e-37

    return [out(h @ w2, [(h, w2, f * E, eh @ w2.abs())]),
            out(da @ w1.t() + db @ w3.t(), [(da, w1.t(), f * E, eda @ w1.t().abs()), (db, w3.t(), f * E, edb @ w3.t().abs())]),
            out(x.t() @ da, [(x.t(), da, m * E, x.t().abs() @ eda)]), out(x.t() @ db, [(x.t(), db, m * E, x.t().abs() @ edb)]),
            out(h.t() @ dy, [(h.t(), dy, m * E, eh.t() @ dy.abs())])]


def step(x, w1, w3, w2, dy):
    from mimir_b200 import tensor as T
    y, kept = T.mlp_gated_fwd(x, w1, w3, w2)
    out = (y,) + tuple(T.mlp_gated_bwd(dy, x, w1, w3, w2, kept))
    T.device_status()
    return out


# one row and one column; extents below, at and past a tile's; rows that are no multiple of 16 bytes; k-blocks dealt out (few rows, many hidden
# columns); several tiles in every direction
SHAPES = [(1, 8, 8, 8), (1, 1, 1, 1), (3, 5, 7, 9), (31, 64, 128, 64), (33, 72, 200, 136), (127, 129, 131, 133), (128, 256, 512, 256),
          (257, 264, 520, 248), (1, 512, 4096, 384), (65, 1000, 3001, 520), (700, 300, 260, 900), (2049, 128, 136, 64)]


@pytest.mark.parametrize("shape,nk", list(itertools.product(SHAPES, [False, True])))
def test_block_and_gradients(shape, nk):
    args = inputs(*shape, nk)
    got = step(*args)
    for name, g, (want, bound), like in zip(("y", "dx", "dw1", "dw3", "dw2"), got, formulas(*args), (None, args[0], *args[1:4])):
        assert g.dtype == BF16 and tuple(g.shape) == tuple(want.shape)
        assert bool(((g.double() - want).abs() <= bound).all()), (name, float(((g.double() - want).abs() / bound).max()))
        if like is not None and like.dim() == 2 and min(like.shape) > 1:
            assert g.stride() == like.stride(), name


@pytest.mark.parametrize("zero", range(4))
def test_empty_extents(zero):
    shape = [24, 40, 56, 72]
    shape[zero] = 0
    args = inputs(*shape, False, std=1.0)
    for g, shape_of in zip(step(*args), (args[4], args[0], *args[1:4])):
        assert g.shape == shape_of.shape and not bool(g.any())


def test_operands_that_start_anywhere_and_are_not_dense():
    m, k, f, n = 70, 96, 160, 88
    args = inputs(m, k, f, n, False, seed=9)
    want = step(*args)

    def moved(t):  # one element past an aligned address
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:].copy_(t.reshape(-1))
        return room[1:].view(t.shape)

    def wide(t):   # rows of a wider matrix
        room = torch.full((t.shape[0], t.shape[1] + 3), float("nan"), dtype=t.dtype, device="cuda")
        room[:, :t.shape[1]] = t
        return room[:, :t.shape[1]]

    for change in (moved, wide):
        for g, w in zip(step(*(change(t) for t in args)), want):
            assert torch.equal(g, w)


def test_same_bits_again_and_on_another_stream():
    args = inputs(130, 512, 2048, 512, True, seed=3)
    want = step(*args)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = step(*args)
    torch.cuda.current_stream().wait_stream(other)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_captured_in_a_graph():
    from mimir_b200 import tensor as T
    args = inputs(100, 256, 768, 264, False, seed=4)
    want = step(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, kept = T.mlp_gated_fwd(*args[:4])
        got = (y,) + tuple(T.mlp_gated_bwd(args[4], *args[:4], kept))
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_infinities_and_nan_stay_in_their_rows():
    args = list(inputs(64, 64, 192, 64, False, seed=5))
    clean = step(*args)
    args[0] = args[0].clone()
    args[0][7, 3], args[0][40, 0] = float("nan"), float("inf")
    y, dx = step(*args)[:2]
    keep = torch.ones(64, dtype=torch.bool, device="cuda")
    keep[[7, 40]] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert bool(y[7].isnan().all())


def test_large_and_small_activations():
    # silu and its derivative where exp overflows (a = -200) and where it vanishes (a = 200)
    x = torch.eye(8, dtype=BF16, device="cuda")
    a = torch.tensor([-200.0, -90.0, -20.0, -1e-3, 0.0, 1e-3, 20.0, 200.0], device="cuda").to(BF16)
    w1, w3, w2 = a.repeat(8, 1).t().contiguous(), torch.full((8, 8), 1.5, device="cuda").to(BF16), torch.eye(8, dtype=BF16, device="cuda")
    args = (x, w1, w3, w2, torch.ones((8, 8), device="cuda").to(BF16))
    for g, (want, bound) in zip(step(*args), formulas(*args)):
        assert bool(((g.double() - want).abs() <= bound).all())


def test_gradient_against_differences():
    """<y, dy> along a step of x and of each weight: the quotient of two forward passes against the gradients. Rounding to bf16 gives each of
    the two sums a noise of 0.6 u of its terms' root sum of squares (the result's own, and as much again from h); six of those, over the
    step, and the quotient's curvature, which the formulas give."""
    from mimir_b200 import tensor as T
    m, k, f, n = 96, 64, 128, 80
    args = list(inputs(m, k, f, n, False, seed=6))
    got = step(*args)
    dy = args[4].double()

    def loss(ts):
        return float((T.mlp_gated_fwd(*ts)[0].double() * dy).sum())

    def exact(ts):
        x, w1, w3, w2 = (t.double() for t in ts)
        a = x @ w1
        return (a * torch.sigmoid(a) * (x @ w3)) @ w2

    y = exact(args[:4])
    noise = 0.6 * U * 2 ** 0.5 * float((y * dy).norm()) * 2 ** 0.5
    for at in range(4):
        direction = torch.sign(got[at + 1].float()) * args[at].float().abs().mean()
        plus, minus = list(args[:4]), list(args[:4])
        plus[at], minus[at] = ((args[at].float() + s * direction / 16).to(BF16) for s in (1, -1))
        delta = plus[at].double() - minus[at].double()
        quotient, slope = loss(plus) - loss(minus), float((got[at + 1].double() * delta).sum())
        curvature = abs(float(((exact(plus) - exact(minus)) * dy).sum()) - float((formulas(*args)[at + 1][0] * delta).sum()))
        allowed = 6 * noise + curvature + U * float((got[at + 1].double() * delta).abs().sum())
        assert abs(slope) > 4 * allowed, "the step says nothing"
        assert abs(quotient - slope) <= allowed, (at, quotient, slope, allowed)


def test_refusals():
    from mimir_b200 import MimkError, _lib
    from mimir_b200 import tensor as T
    x, w1, w3, w2, dy = inputs(16, 32, 48, 24, False)
    y, kept = T.mlp_gated_fwd(x, w1, w3, w2)
    with pytest.raises(ValueError, match="contracting dims"):
        T.mlp_gated_fwd(x, w1, w3, w2[:40])
    with pytest.raises(ValueError, match="rank-2"):
        T.mlp_gated_fwd(x[None], w1, w3, w2)
    with pytest.raises(ValueError, match="storage layout"):
        T.mlp_gated_fwd(x, w1, w3.t().contiguous().t(), w2)
    with pytest.raises(TypeError):
        T.mlp_gated_fwd(x, w1.float(), w3, w2)
    with pytest.raises(MimkError) as e:
        T.mlp_gated_fwd(x.float(), w1.float(), w3.float(), w2.float())
    assert e.value.status == 4                              # MIMK_E_DTYPE: bf16 only, as mlp_gated
    with pytest.raises(ValueError, match="CUDA tensors only"):
        T.mlp_gated_fwd(x.cpu(), w1, w3, w2)
    with pytest.raises(ValueError, match="result's shape"):
        T.mlp_gated_bwd(dy[:8], x, w1, w3, w2, kept)
    with pytest.raises(ValueError, match="other extents"):
        T.mlp_gated_bwd(dy[:8], x[:8], w1, w3, w2, kept)
    with pytest.raises(TypeError):
        T.mlp_gated_bwd(dy.float(), x, w1, w3, w2, kept)
    # the C entry points: a workspace that is missing, too small or unaligned; kept and results that are missing
    import ctypes as C
    d, held = T._mlp_train_desc(x, w1, w3, w2)
    dx, g1, g3, g2 = torch.empty_like(x), torch.empty_like(w1), torch.empty_like(w3), torch.empty_like(w2)
    d.dy, d.dx, d.dw1, d.dw3, d.dw2 = (t.data_ptr() for t in (dy, dx, g1, g3, g2))
    lib, need = _lib.lib(), C.c_uint64()
    assert lib.mimk_mlp_gated_bwd(C.byref(d), None) == 1
    d.kept = kept.buffer.data_ptr()
    assert lib.mimk_mlp_gated_train_sizes(C.byref(d), None, None, C.byref(need)) == 0 and need.value > 0
    assert lib.mimk_mlp_gated_bwd(C.byref(d), None) == 9
    room = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = room.data_ptr(), need.value - 1
    assert lib.mimk_mlp_gated_bwd(C.byref(d), None) == 9
    d.workspace, d.workspace_bytes = room.data_ptr() + 4, need.value
    assert lib.mimk_mlp_gated_bwd(C.byref(d), None) == 3
    d.dw3 = None
    assert lib.mimk_mlp_gated_bwd(C.byref(d), None) == 1
    d.m = -1
    assert lib.mimk_mlp_gated_fwd(C.byref(d), None) == 1
