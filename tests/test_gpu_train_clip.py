"""Norm and clipping of a list of gradients against 64 bits, through the public operators.

Tolerances. Up to 16 squares are summed in f32 (16 roundings of 2^-24 at most), everything beyond in f64: the norm is within 2^-20 of itself,
with its own rounding. A scaled value is rounded once more: 2^-8 of itself as bf16 (u), 2^-23 as F32.
"""
import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def reference(grads, limit, eps=1e-6):
    norm = sum(float(g.double().square().sum()) for g in grads) ** 0.5
    c = min(1.0, limit / (norm + eps))
    return norm, [g.double() * c for g in grads]


def holds(norm, got, want_norm, want):
    assert abs(float(norm) - want_norm) <= 2.0 ** -20 * want_norm
    for g, w in zip(got, want):
        u = 2.0 ** -8 if g.dtype == BF16 else 2.0 ** -23
        assert bool(((g.double() - w).abs() <= (u + 2.0 ** -20) * w.abs() + (1e-40 if g.dtype == BF16 else 1e-44)).all())


def some(sizes, dtypes, seed=0, std=1.0):
    return [randn((s,), seed + i, std, dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16)])
@pytest.mark.parametrize("limit", [0.5, 1e6, 0.0])
@pytest.mark.parametrize("sizes", [[1], [0], [0, 3, 0], [7, 8, 9, 15, 16, 17], [16383, 16384, 16385, 1], [300000, 2, 5000]])
def test_clipping(sizes, limit, dtypes):
    from mimir_b200 import tensor as T
    grads = some(sizes, dtypes)
    want_norm, want = reference(grads, limit)
    norm = T.grad_norm(grads)
    assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - want_norm) <= 2.0 ** -20 * want_norm
    before = [g.clone() for g in grads]
    out = [torch.full_like(g, float("nan")) for g in grads]
    holds(T.clip_grad_norm(grads, limit, out=out), out, want_norm, want)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    holds(T.clip_grad_norm(grads, limit), grads, want_norm, want)
    assert all(torch.equal(g, o) for g, o in zip(grads, out))
    if limit == 1e6:
        assert all(torch.equal(g, b) for g, b in zip(grads, before))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1])
def test_packed_at_any_offset(dtype, shift):
    from mimir_b200 import tensor as T
    sizes = [(7 * i * i) % 5003 + 1 for i in range(1500)]      # more than one table, every alignment
    flat = randn((sum(sizes),), 3, 1.0, dtype)
    room = torch.empty((flat.numel() + 1,), dtype=dtype, device="cuda")
    out = room[shift:shift + flat.numel()]                     # shift 1: results that lie otherwise than the gradients
    want_norm, (want,) = reference([flat], 2.0)
    holds(T.clip_grad_norm(list(flat.split(sizes)), 2.0, out=list(out.split(sizes))), [out], want_norm, [want])


def test_neighbours_are_left_alone():
    from mimir_b200 import tensor as T
    for dtype in (F32, BF16):
        for at, size in ((1, 1), (3, 40), (5, 70001), (8, 16384)):
            room = torch.ones((size + 16,), dtype=dtype, device="cuda")
            out = torch.full((size + 16,), 5.0, dtype=dtype, device="cuda")
            norm = T.clip_grad_norm([room[at:at + size]], 0.25, out=[out[at:at + size]])
            assert abs(float(norm) - size ** 0.5) <= 2.0 ** -20 * size ** 0.5
            assert bool((out[:at] == 5).all()) and bool((out[at + size:] == 5).all()) and bool((out[at:at + size] < 0.3).all())


def test_values_whose_squares_are_no_f32():
    from mimir_b200 import tensor as T
    for dtype in (F32, BF16):
        for value in (1e-38, 1e-30, 1e-20, 1e20, 1e30, 3e38):
            g = torch.full((1000,), value, device="cuda").to(dtype)
            want_norm, want = reference([g], 0.5 * float(g[0]), eps=0.0)
            if want_norm < 3.4e38:
                out = torch.empty_like(g)
                holds(T.clip_grad_norm([g], 0.5 * float(g[0]), eps=0.0, out=[out]), [out], want_norm, want)
            else:
                assert bool(T.grad_norm([g]).isinf())


def test_values_that_are_not_finite():
    from mimir_b200 import tensor as T
    for dtype in (F32, BF16):
        a, b = randn((5000,), 1, 1.0, dtype), randn((33,), 2, 1.0, dtype)
        a[77] = float("inf")
        out = [torch.empty_like(a), torch.empty_like(b)]
        assert bool(T.clip_grad_norm([a, b], 1.0, out=out).isinf())
        assert bool(out[0][77].isnan()) and int(out[0].isnan().sum()) == 1 and not bool(out[1].any())
        b[3] = float("nan")
        assert bool(T.clip_grad_norm([a, b], 1.0).isnan()) and bool(a.isnan().all()) and bool(b.isnan().all())


def test_layouts_views_and_an_empty_list():
    from mimir_b200 import tensor as T
    w = randn((40, 56), 1, 1.0, BF16)
    grads = [w.t(), randn((3, 4, 5), 2).permute(2, 0, 1), randn((), 3)]
    want_norm, want = reference(grads, 1.0)
    holds(T.clip_grad_norm(grads, 1.0), grads, want_norm, want)
    assert float(T.grad_norm([])) == 0 and float(T.clip_grad_norm([], 1.0)) == 0
    wide = randn((8, 16), 4)
    for bad in (wide[:, :5], wide[:, ::2], wide[:1].expand(8, 16)):
        with pytest.raises(ValueError, match="dense"):
            T.grad_norm([bad])


def test_same_bits_again_and_on_another_stream_and_in_a_graph():
    from mimir_b200 import tensor as T
    grads = some([123457, 999, 70000], (F32, BF16))
    out = [torch.empty_like(g) for g in grads]
    norm = T.clip_grad_norm(grads, 1.0, out=out)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        second = [torch.empty_like(g) for g in grads]
        assert torch.equal(T.clip_grad_norm(grads, 1.0, out=second), norm)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(out, second))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = T.clip_grad_norm(grads, 1.0, out=second)
    for g in grads:
        g.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert abs(float(again) - 2 * float(norm)) <= 2.0 ** -19 * float(again)


def test_refusals():
    from mimir_b200 import _lib
    from mimir_b200 import tensor as T
    g = randn((64,), 1)
    with pytest.raises(TypeError, match="F32 or BF16"):
        T.grad_norm([g.half()])
    with pytest.raises(TypeError, match="same element type"):
        T.clip_grad_norm([g], 1.0, out=[g.to(BF16)])
    with pytest.raises(ValueError, match="one result"):
        T.clip_grad_norm([g], 1.0, out=[])
    with pytest.raises(ValueError, match="same shape"):
        T.clip_grad_norm([g], 1.0, out=[g[:32]])
    with pytest.raises(ValueError, match="CUDA tensors only"):
        T.grad_norm([g.cpu()])
    for limit, eps in ((-1.0, 0.0), (float("nan"), 0.0), (1.0, -1e-6)):
        with pytest.raises(ValueError, match="at least 0"):
            T.clip_grad_norm([g], limit, eps=eps)
    import ctypes as C
    lib, need = _lib.lib(), C.c_uint64()
    assert lib.mimk_clip_grads_workspace(1, C.byref(need)) == 0
    ins, n, dt = (C.c_void_p * 1)(g.data_ptr()), (C.c_int64 * 1)(64), (C.c_int32 * 1)(_lib.F32)
    norm, room = torch.zeros((), device="cuda"), torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    assert lib.mimk_grad_norm(ins, n, dt, 1, norm.data_ptr(), None, 0, None) == 9
    assert lib.mimk_grad_norm(ins, n, dt, 1, norm.data_ptr(), room.data_ptr(), need.value - 1, None) == 9
    assert lib.mimk_grad_norm(ins, n, dt, 1, norm.data_ptr(), room.data_ptr() + 4, need.value, None) == 3
    ins[0] = g.data_ptr() + 2
    assert lib.mimk_grad_norm(ins, n, dt, 1, norm.data_ptr(), room.data_ptr(), need.value, None) == 3
