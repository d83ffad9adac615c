"""Cross-entropy of a linear layer against its formulas in 64 bits, through the public operators.

Tolerances. A logit is a sum of d products in f32: at most d 2^-23 of the product of the magnitudes off (e_l), and 2^-20 of it more for F32 operands,
whose products have 21 bits. log sum exp moves by no more than the largest e_l of its row, exp and log by some units of 2^-22. The factor
p = g (softmax - onehot) moves by softmax (e_l + e_lse), and for bf16 it is rounded (u = 2^-8); gradients are sums of products with it, and for bf16
they are rounded again.
"""
import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -22
BF16, F32 = torch.bfloat16, torch.float32
IGNORED = -100


def inputs(n, d, v, dtype, nk, seed=0, masked=0.0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 100)
    t = torch.randint(0, v, (n,), generator=g)
    if masked:
        t[torch.rand((n,), generator=g) < masked] = IGNORED
    x = randn((n, d), seed, 1.0, dtype)
    w = randn((v, d), seed + 1, spread * d ** -0.5, dtype).t() if nk else randn((d, v), seed + 1, spread * d ** -0.5, dtype)
    return x, w, t.cuda()


def formulas(x, w, t, g=None, mean=True):
    """losses, lse, dx, dw and a bound of each one's error, in 64 bits. g: the gradient that arrives at each loss."""
    bf16 = x.dtype == BF16
    x, w = x.double(), w.double()
    n, d, v = *x.shape, w.shape[1]
    kept = (t >= 0) & (t < v)
    x = torch.where(kept[:, None], x, 0.0)
    at = torch.where(kept, t.long(), 0)[:, None]
    l, mag = x @ w, x.abs() @ w.abs()
    el = mag * (d * E / 2 + (0 if bf16 else 2.0 ** -20))
    lse = torch.logsumexp(l, 1)
    elsx = el.max(1).values + 8 * E + E * lse.abs()
    loss = lse - l.gather(1, at)[:, 0]
    eloss = elsx + el.gather(1, at)[:, 0] + E * (loss.abs() + l.gather(1, at)[:, 0].abs())
    each = kept.double() * (1.0 if g is None else g)
    if mean:
        each = each / max(int(kept.sum()), 1)
    p = torch.exp(l - lse[:, None])
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    dl = each[:, None] * (p - one)
    edl = each.abs()[:, None] * (p * ((el + elsx[:, None]) * 1.01 + E * (8 + (l - lse[:, None]).abs())) + E * one) + 4 * E * dl.abs()
    if bf16:
        edl = edl + U * dl.abs()
    terms = 0 if bf16 else 2.0 ** -20
    dx, dw = dl @ w.t(), x.t() @ dl
    edx = (edl @ w.t().abs()) + (v * E + terms) * (dl.abs() @ w.t().abs()) + (U if bf16 else E) * dx.abs()
    edw = (x.t().abs() @ edl) + (n * E + terms) * (x.t().abs() @ dl.abs()) + (U if bf16 else E) * dw.abs()
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    return [(torch.where(kept, loss, zero), eloss), (torch.where(kept, lse, zero), elsx), (dx, edx * 1.02 + 1e-37), (dw, edw * 1.02 + 1e-37)], kept


def near(got, want, bound):
    return bool(((got.double() - want).abs() <= bound).all())


# one row, one class, one feature; extents below, at and past a tile's; rows of no whole 16 bytes; several tiles in every direction; k-blocks dealt
# out (few rows, many classes)
SHAPES = [(1, 8, 8), (1, 1, 1), (3, 5, 7), (64, 64, 256), (33, 72, 257), (127, 129, 1000), (300, 64, 513), (5, 128, 20000), (257, 136, 3001), (1000, 40, 72)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("masked", [0.0, 0.4])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(shape, masked, nk, dtype):
    from mimir_b200 import tensor as T
    x, w, t = inputs(*shape, dtype, nk, masked=masked)
    ignore = IGNORED if masked else None
    want, kept = formulas(x, w, t)
    losses, lse = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="none", return_lse=True)
    assert losses.dtype == lse.dtype == F32
    assert near(losses, *want[0]) and near(lse, *want[1])
    count = max(int(kept.sum()), 1)
    for reduction, over in (("mean", count), ("sum", 1)):
        got = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction=reduction)
        assert got.dim() == 0 and abs(float(got) - float(want[0][0].sum()) / over) <= float(want[0][1][kept].sum()) / over + 1e-37 + E * abs(float(got))
    loss, dx, dw = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=ignore)
    assert torch.equal(loss, T.linear_cross_entropy(x, w, t, ignore_index=ignore))
    assert dx.dtype == dw.dtype == dtype and dx.shape == x.shape and dw.shape == w.shape
    assert min(w.shape) == 1 or dw.stride() == w.stride()
    assert near(dx, *want[2]) and near(dw, *want[3])
    again = T.linear_cross_entropy_grad(x, w, t, lse, ignore_index=ignore)
    assert near(again[0], *want[2]) and near(again[1], *want[3])
    T.device_status()


@pytest.mark.parametrize("dtype,shape", [(BF16, (70000, 16, 8300)), (F32, (1500, 12, 131072))])
@pytest.mark.parametrize("nk", [False, True])
def test_several_pieces(dtype, shape, nk):
    from mimir_b200 import tensor as T
    x, w, t = inputs(*shape, dtype, nk, masked=0.2)
    _, dx, dw = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED, reduction="sum")
    lse = T.linear_cross_entropy(x, w, t, ignore_index=IGNORED, reduction="none", return_lse=True)[1]
    total, bound = torch.zeros(w.shape, dtype=torch.float64, device="cuda"), torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    for i in range(0, shape[0], 5000):
        want, _ = formulas(x[i:i + 5000], w, t[i:i + 5000], mean=False)
        assert near(lse[i:i + 5000], *want[1]) and near(dx[i:i + 5000], *want[2])
        total += want[3][0]
        bound += want[3][1]
    # (the bounds of the parts hold their roundings; sums over all rows in f32 add n E of the magnitudes at most, as those do for their own)
    assert near(dw, total, bound * (1 + shape[0] / 5000))


@pytest.mark.parametrize("shape", [(1, 64, 1000), (2, 8, 5), (3, 136, 5001), (4, 4096, 778), (2, 4096, 40000), (1, 16384, 130), (4, 4104, 130)])
@pytest.mark.parametrize("masked", [0.0, 0.6])
def test_scoring_a_few_rows(shape, masked):
    from mimir_b200 import tensor as T
    x, w, t = inputs(*shape, BF16, True, seed=11, masked=masked)
    ignore = IGNORED if masked else None
    want, kept = formulas(x, w, t)
    losses, lse = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="none", return_lse=True)
    assert near(losses, *want[0]) and near(lse, *want[1])
    total = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="sum")
    assert abs(float(total) - float(want[0][0].sum())) <= float(want[0][1][kept].sum()) + 1e-37 + E * abs(float(total))
    if masked == 0.0:
        w = w.clone(memory_format=torch.preserve_format)
        w[:, shape[2] // 2:] = float("-inf") * torch.sign(x[0]).to(w.dtype)[:, None]      # (row 0's scores of half the classes are -inf)
        t = t % max(shape[2] // 2, 1)
        losses = T.linear_cross_entropy(x, w, t, reduction="none")
        half, _ = formulas(x[:1], w[:, :shape[2] // 2].t().contiguous().t(), t[:1])
        assert abs(float(losses[0]) - float(half[0][0])) <= float(half[0][1])


def test_gradients_that_arrive_and_targets_of_32_bits():
    from mimir_b200 import tensor as T
    x, w, t = inputs(90, 48, 300, BF16, True, masked=0.3)
    g = randn((90,), 7)
    lse = T.linear_cross_entropy(x, w, t, ignore_index=IGNORED, return_lse=True)[1]
    want, _ = formulas(x, w, t, g.double(), mean=False)
    for targets in (t, t.int()):
        dx, dw = T.linear_cross_entropy_grad(x, w, targets, lse, ignore_index=IGNORED, reduction="none", dloss=g)
        assert near(dx, *want[2]) and near(dw, *want[3])
    want, _ = formulas(x, w, t, 0.25)
    dx, dw = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED, dloss=torch.tensor(0.25, device="cuda"))[1:]
    assert near(dx, *want[2]) and near(dw, *want[3])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_without_a_target_are_not_read(dtype):
    from mimir_b200 import tensor as T
    for rows in (slice(0, 80), slice(0, 40), slice(37, 80), slice(10, 11)):
        x, w, t = inputs(80, 64, 500, dtype, False, seed=2)
        t[rows] = IGNORED
        clean = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED)
        bad = x.clone()
        bad[rows] = float("nan")
        for a, b in zip(clean, T.linear_cross_entropy_with_grad(bad, w, t, ignore_index=IGNORED)):
            assert torch.equal(a, b) and not bool(a.isnan().any())
        assert not bool(clean[1][rows].any())
        assert not bool(T.linear_cross_entropy(bad, w, t, ignore_index=IGNORED, reduction="none")[rows].any())
        if rows == slice(0, 80):
            assert float(clean[0]) == 0 and not bool(clean[2].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ignore", [None, IGNORED])
def test_targets_that_are_no_class(dtype, ignore):
    from mimir_b200 import MimkError
    from mimir_b200 import tensor as T
    x, w, t = inputs(70, 64, 300, dtype, True, seed=3)
    want = T.linear_cross_entropy_with_grad(torch.cat([x[:5], x[6:]]), w, torch.cat([t[:5], t[6:]]), reduction="sum")
    for wrong in (300, -1, 1 << 40):
        t[5] = wrong
        losses = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="none")
        with pytest.raises(MimkError) as e:
            T.device_status()
        assert e.value.status == 2                           # MIMK_E_SHAPE
        assert bool(losses[5].isnan()) and int(losses.isnan().sum()) == 1
        loss, dx, dw = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=ignore, reduction="sum")
        assert bool(loss.isnan()) and not bool(dx[5].any())
        tol = 1e-2 if dtype == BF16 else 1e-5                # (another order of the rows: other roundings)
        assert float((dw - want[2]).norm() / want[2].norm()) <= tol and float((dx[6:] - want[1][5:]).norm() / want[1].norm()) <= tol
        with pytest.raises(MimkError):
            T.device_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_far_apart_and_not_finite(dtype):
    from mimir_b200 import tensor as T
    # the logits are the row of w that x picks: far apart, all equal, and with infinities
    x = torch.eye(4, device="cuda").to(dtype)
    w = torch.zeros((4, 300), device="cuda")
    w[0, 7], w[0, 8], w[1] = 2.0 ** 14, -2.0 ** 14, -3.0e4
    w[2, 17:] = -80.0
    w = w.to(dtype)
    t = torch.tensor([7, 0, 250, 3], device="cuda")
    losses, lse = T.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    want, _ = formulas(x, w, t)
    assert near(losses, *want[0]) and near(lse, *want[1])
    assert bool(torch.isfinite(losses).all())
    dx, dw = T.linear_cross_entropy_with_grad(x, w, t)[1:]
    want[2][1].add_(1e-3 * want[2][0].abs())                 # (terms of 2^14 cancel: f32 sums of them)
    assert near(dw, *want[3])
    # a class whose score is -inf has no weight (x is all ones here: 0 inf would be NaN)
    x = torch.ones((2, 4), device="cuda").to(dtype)
    w = randn((4, 600), 5, 1.0, dtype)
    w[:, :256] = float("-inf")
    losses, lse = T.linear_cross_entropy(x, w, torch.tensor([300, 599], device="cuda"), reduction="none", return_lse=True)
    want, _ = formulas(x, w[:, 256:].contiguous(), torch.tensor([44, 343], device="cuda"))
    assert near(losses, *want[0]) and near(lse, *want[1])
    # NaN stays in its row
    x = randn((40, 32), 6, 1.0, dtype)
    w, t = randn((32, 500), 8, 1.0, dtype), torch.arange(40, device="cuda")
    clean = T.linear_cross_entropy(x, w, t, reduction="none")
    x[9, 4] = float("nan")
    losses = T.linear_cross_entropy(x, w, t, reduction="none")
    keep = torch.arange(40, device="cuda") != 9
    assert bool(losses[9].isnan()) and torch.equal(losses[keep], clean[keep])


def test_no_rows_and_leading_axes():
    from mimir_b200 import tensor as T
    for dtype in (BF16, F32):
        x, w, t = inputs(24, 32, 100, dtype, True)
        loss, dx, dw = T.linear_cross_entropy_with_grad(x[:0], w, t[:0])
        assert float(loss) == 0 and dx.shape == (0, 32) and not bool(dw.any())
        assert T.linear_cross_entropy(x[:0], w, t[:0], reduction="none").shape == (0,)
        want = T.linear_cross_entropy_with_grad(x, w, t)
        got = T.linear_cross_entropy_with_grad(x.view(2, 3, 4, 32), w, t.view(2, 3, 4))
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1].view(24, 32)) and torch.equal(want[2], got[2])
        assert T.linear_cross_entropy(x.view(4, 6, 32), w, t.view(4, 6), reduction="none").shape == (4, 6)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_operands_that_start_anywhere_and_are_not_dense(dtype):
    from mimir_b200 import tensor as T
    x, w, t = inputs(70, 96, 304, dtype, False, seed=4, masked=0.2)
    want = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED)

    def moved(a):
        room = torch.empty(a.numel() + 1, dtype=a.dtype, device="cuda")
        room[1:].copy_(a.reshape(-1))
        return room[1:].view(a.shape)

    def wide(a):
        room = torch.zeros((a.shape[0], a.shape[1] + 3) if a.dim() == 2 else (a.shape[0], 2), dtype=a.dtype, device="cuda")
        view = room[:, :a.shape[1]] if a.dim() == 2 else room[:, 0]
        view.copy_(a)
        return view

    for change in (moved, wide):
        for g, h in zip(T.linear_cross_entropy_with_grad(change(x), change(w), change(t), ignore_index=IGNORED), want):
            assert torch.equal(g, h) or (dtype == F32 and float((g - h).norm() / h.norm()) <= 1e-5)  # (f32 products choose a kernel by alignment)


def test_same_bits_again_and_on_another_stream_and_in_a_graph():
    from mimir_b200 import tensor as T
    x, w, t = inputs(200, 128, 5000, BF16, True, seed=5, masked=0.2)
    want = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED)
    t.copy_(torch.roll(t, 3))     # other rows without a target: how many there are is found out on the device
    want = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=IGNORED)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_against_differences(dtype):
    """The loss at x + s and x - s against <dx, 2 s>, s a step along the gradient's signs; likewise for w. The losses' own bounds, and the quotient's
    curvature, which the formulas give, are allowed for."""
    from mimir_b200 import tensor as T
    x, w, t = inputs(60, 64, 400, dtype, False, seed=6)
    grads = T.linear_cross_entropy_with_grad(x, w, t, reduction="sum")[1:]
    for at in range(2):
        ends = []
        for sign in (1, -1):
            moved = [x, w]
            moved[at] = (moved[at].float() + sign * torch.sign(grads[at].float()) * moved[at].float().abs().mean() / 8).to(dtype)
            ends.append(moved)
        delta = ends[0][at].double() - ends[1][at].double()
        losses = [float(T.linear_cross_entropy(*e, t, reduction="sum")) for e in ends]
        exact = [formulas(*e, t, mean=False)[0] for e in ends]
        want = formulas(x, w, t, mean=False)[0][2 + at]
        slope, true = float((grads[at].double() * delta).sum()), float((want[0] * delta).sum())
        curvature = abs(float(exact[0][0][0].sum() - exact[1][0][0].sum()) - true)
        allowed = curvature + float((want[1] * delta.abs()).sum()) + float(exact[0][0][1].sum() + exact[1][0][1].sum())
        assert abs(slope) > 4 * allowed, "the step says nothing"
        assert abs(losses[0] - losses[1] - slope) <= allowed


def test_refusals():
    from mimir_b200 import MimkError, _lib
    from mimir_b200 import tensor as T
    x, w, t = inputs(16, 32, 50, BF16, False)
    with pytest.raises(ValueError, match="contracting dims"):
        T.linear_cross_entropy(x, w[:16], t)
    with pytest.raises(ValueError, match="one target"):
        T.linear_cross_entropy(x, w, t[:8])
    with pytest.raises(ValueError, match="reduction"):
        T.linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(TypeError, match="one element type"):
        T.linear_cross_entropy(x, w.float(), t)
    with pytest.raises(TypeError, match="I32 or I64"):
        T.linear_cross_entropy(x, w, t.float())
    with pytest.raises(TypeError):
        T.linear_cross_entropy(x.half(), w.half(), t)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        T.linear_cross_entropy(x, w, t.cpu())
    with pytest.raises(ValueError, match="lse"):
        T.linear_cross_entropy_grad(x, w, t, torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError, match="dloss"):
        T.linear_cross_entropy_grad(x, w, t, torch.zeros(16, device="cuda"), dloss=torch.zeros(16, device="cuda"))
    with pytest.raises(MimkError) as e:
        T.linear_cross_entropy(x[:, :0], w[:0], t)           # rows, and no feature
    assert e.value.status == 2
    import ctypes as C
    d = _lib.LinearCeDesc()
    loss, room = torch.zeros((), device="cuda"), torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    d.n, d.d, d.v, d.x, d.w, d.targets, d.loss = 16, 32, 50, x.data_ptr(), w.data_ptr(), t.data_ptr(), loss.data_ptr()
    d.dtype, d.target_dtype, d.reduction = _lib.BF16, _lib.I64, _lib.REDUCTION_MEAN
    lib, need = _lib.lib(), C.c_uint64()
    assert lib.mimk_linear_ce_workspace(C.byref(d), 1, 0, C.byref(need)) == 0 and 0 < need.value < room.numel()
    assert lib.mimk_linear_ce_fwd(C.byref(d), None) == 9
    d.workspace, d.workspace_bytes = room.data_ptr(), need.value - 1
    assert lib.mimk_linear_ce_fwd(C.byref(d), None) == 9
    d.workspace, d.workspace_bytes = room.data_ptr() + 8, need.value
    assert lib.mimk_linear_ce_fwd(C.byref(d), None) == 3
    d.workspace = room.data_ptr()
    assert lib.mimk_linear_ce_fwd_bwd(C.byref(d), None) == 1  # no dx, no dw
    assert lib.mimk_linear_ce_bwd(C.byref(d), None) == 1      # no lse
    d.loss = None
    assert lib.mimk_linear_ce_fwd(C.byref(d), None) == 1
