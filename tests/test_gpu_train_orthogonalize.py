"""The orthogonalised update against its definition in 64 bits, through the public operator.

Tolerances. What the operator rounds on the way is known: the values of A and of q A + r A^2 off their diagonals and those of X as an operand to 11 bits (each off by at most 2^-11 of
itself), X itself to 22 (2^-22; as an f32 and twice an f16, with what lies below 2^-33), and the products' sums, which tensor cores cut off where f32 rounds (2^-22 of the magnitudes' sum, as
a bound for rows of these lengths). How such errors grow through the steps depends on the matrix, so the oracle makes them: the definition in 64 bits with independent relative errors, uniform to
those bounds, in the same places, eight times over. The roundings of one matrix are one more such draw, each error smaller than the bound that the oracle draws to (half a step, whose mean over a binade
is three quarters of the bound), so that the 2-norm of the whole deviation lies within the largest of eight draws but for the spread of a 2-norm of few values: twice the largest is allowed, and to that the
rounding of the result to bf16, 2^-8 of each value. For single values: eight times the root mean square of the deviation (beyond what 10^7 values of a normal spread reach), and the rounding."""
import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
STEPS = ((3.4445, -4.7750, 2.0315),) * 5


def matrix(kind, shape, seed=0):
    m, n = shape[-2:]
    x = randn(shape, seed)
    if kind == "falling":
        k = min(m, n)
        left, right = randn((*shape[:-2], m, k), seed + 1), randn((*shape[:-2], k, n), seed + 2)
        x = (left * torch.logspace(0, -2.5, k, device="cuda")) @ right
    if kind == "rank":
        x = randn((*shape[:-2], m, 2), seed + 1) @ randn((*shape[:-2], 2, n), seed + 2) + 0.05 * x
    return x


def oracle(x, steps=STEPS, eps=1e-7, seed=None):
    """[..., m, n] in 64 bits; with a seed, with errors of the operator's roundings."""
    x = x.double()
    m, n = x.shape[-2:]
    g = None if seed is None else torch.Generator(device="cuda").manual_seed(seed)
    off = lambda t, u: t if g is None else t * (1 + u * (2 * torch.rand(t.shape, generator=g, device="cuda", dtype=torch.float64) - 1))  # noqa: E731
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    x = x if m <= n else x.mT
    for p, q, r in steps:
        x = off(x, 2.0 ** -22)
        operand = off(x, 2.0 ** -11)
        a = off(operand @ operand.mT, 2.0 ** -22)
        d = torch.diagonal(a, dim1=-2, dim2=-1)
        o = off(a - torch.diag_embed(d), 2.0 ** -11)
        b = q * (o + torch.diag_embed(d)) + r * off(o @ o + (d.unsqueeze(-1) + d.unsqueeze(-2)) * o + torch.diag_embed(d * d), 2.0 ** -22)
        e = torch.diagonal(b, dim1=-2, dim2=-1)
        x = (p + e).unsqueeze(-1) * x + off(off(b - torch.diag_embed(e), 2.0 ** -11) @ operand, 2.0 ** -22)
    return x if m <= n else x.mT


def check(x, got, steps=STEPS, eps=1e-7, scale=1.0):
    assert got.dtype == BF16 and got.shape == x.shape
    for one, out in zip(x.reshape(-1, *x.shape[-2:]), got.reshape(-1, *x.shape[-2:])):
        want = oracle(one, steps, eps)
        off = 2 * max(float((oracle(one, steps, eps, s) - want).norm()) for s in range(8))
        rounding = want.abs() * 2.0 ** -8 * 1.01
        diff = (out.double() / scale - want).abs()
        assert float(diff.norm()) <= off + float(rounding.norm()), (float(diff.norm() / want.norm()), off / float(want.norm()))
        assert bool((diff <= 8 * off / want.numel() ** 0.5 + rounding).all())


# one value, one row, one column; below, at and past a tile's and a pair's; rows of no whole 16 bytes, either way; several tiles in each direction
SHAPES = [(1, 1), (1, 8), (9, 1), (2, 3), (7, 5), (8, 64), (31, 33), (64, 64), (64, 65), (127, 129), (129, 127), (128, 128), (128, 520), (520, 128), (129, 136), (136, 257), (255, 703),
          (703, 255), (256, 256), (257, 1000), (1000, 264), (513, 515), (640, 641), (30, 5000), (5000, 30), (1300, 1100)]


@pytest.mark.parametrize("shape", SHAPES)
def test_random_matrices(shape):
    from mimir_b200 import tensor as T
    for dtype in (F32, BF16):
        x = matrix("random", shape).to(dtype)
        check(x, T.orthogonalize(x))
    T.device_status()


@pytest.mark.parametrize("shape", [(16, 40), (64, 64), (100, 300), (300, 100), (256, 704), (520, 520), (1100, 640)])
@pytest.mark.parametrize("kind", ["falling", "rank"])
def test_falling_singular_values(kind, shape):
    from mimir_b200 import tensor as T
    x = matrix(kind, shape)
    check(x, T.orthogonalize(x))
    check(x.to(BF16), T.orthogonalize(x.to(BF16)))
    T.device_status()


def test_large():
    """Tiles of pairs of SMs in every product."""
    from mimir_b200 import tensor as T
    for shape in ((2600, 2904), (2904, 2600)):
        x = matrix("falling", shape, 3)
        check(x, T.orthogonalize(x))
    T.device_status()


@pytest.mark.parametrize("shape", [(5, 64, 64), (2, 3, 24, 40), (70, 128, 128), (3, 300, 200), (9, 13, 7), (2, 1, 5), (150, 40, 264)])
def test_stacks(shape):
    from mimir_b200 import tensor as T
    x = matrix("random", shape, 4)
    got = T.orthogonalize(x)
    check(x[..., :2, :, :] if len(shape) == 4 else x[:3], got[..., :2, :, :] if len(shape) == 4 else got[:3])
    # a matrix comes out the same alone
    flat, out = x.reshape(-1, *shape[-2:]), got.reshape(-1, *shape[-2:])
    assert torch.equal(T.orthogonalize(flat[-1]), out[-1]) and torch.equal(T.orthogonalize(flat[:1])[0], out[0])


def test_lists():
    from mimir_b200 import tensor as T
    xs = [matrix("random", s, 5 + i).to(t) for i, (s, t) in enumerate([((64, 96), F32), ((3, 64, 96), F32), ((96, 64), BF16), ((64, 96), BF16), ((64, 96), F32), ((0, 96), F32), ((2, 0, 4, 4), F32)])]
    got = T.orthogonalize(xs)
    assert isinstance(got, list) and len(got) == len(xs)
    for x, g in zip(xs, got):
        assert g.shape == x.shape and g.dtype == BF16 and torch.equal(g, T.orthogonalize(x))
    assert T.orthogonalize([]) == []
    assert torch.equal(T.orthogonalize((xs[0],))[0], got[0])


def test_more_matrices_than_one_launch_takes():
    from mimir_b200 import tensor as T
    x = matrix("random", (2100, 9, 12), 6)
    got = T.orthogonalize(x)
    for i in (0, 1023, 1024, 2047, 2048, 2099):
        assert torch.equal(got[i], T.orthogonalize(x[i]))


def test_more_than_the_buffer_holds():
    """Matrices of 8 x 4000 x 4000 bytes and more, of which eight share a buffer of 1 GiB."""
    from mimir_b200 import tensor as T
    x = torch.randn((8, 4000, 3992), device="cuda", generator=torch.Generator(device="cuda").manual_seed(7), dtype=BF16)
    got = T.orthogonalize(x, steps=2)
    assert torch.equal(got[7], T.orthogonalize(x[7], steps=2)) and torch.equal(got[0], T.orthogonalize(x[0], steps=2))
    T.device_status()


def test_transposed_views_and_other_strides():
    from mimir_b200 import tensor as T
    x = matrix("random", (96, 200), 8)
    want = T.orthogonalize(x)
    got = T.orthogonalize(x.t())
    assert got.shape == (200, 96) and got.stride() == x.t().stride() and torch.equal(got, want.t())
    wide = torch.full((96, 203), float("nan"), device="cuda")
    wide[:, :200] = x
    assert torch.equal(T.orthogonalize(wide[:, :200]), want)
    room = torch.empty(96 * 200 + 1, device="cuda")
    room[1:].copy_(x.reshape(-1))
    check(x, T.orthogonalize(room[1:].view(96, 200)))
    stack = matrix("random", (4, 40, 56), 9)
    assert torch.equal(T.orthogonalize(stack.mT), T.orthogonalize(stack).mT)
    assert torch.equal(T.orthogonalize(stack[::2]), T.orthogonalize(stack)[::2])


def test_other_steps():
    from mimir_b200 import tensor as T
    x = matrix("falling", (60, 90), 10)
    for steps, coefficients in ((1, (1.5, -0.5, 0.0)), (12, (1.5, -0.5, 0.0)), (3, (1.875, -1.25, 0.375)), (2, ((3.4445, -4.775, 2.0315), (1.5, -0.5, 0.0))), (2, (0.5, 0.0, 0.0)), (1, (-1.0, 0.25, 0.25))):
        each = coefficients if isinstance(coefficients[0], tuple) else (coefficients,) * steps
        check(x, T.orthogonalize(x, steps=steps, coefficients=coefficients), each)
    check(x, T.orthogonalize(x, scale=-0.25), scale=-0.25)
    check(x * 1e-3, T.orthogonalize(x * 1e-3, eps=0.5), eps=0.5)


@pytest.mark.parametrize("factor", [1e-38, 1e-30, 1e-12, 1e12, 1e30, 1e36])
def test_matrices_of_any_size(factor):
    """The result does not depend on a factor, however large or small, where eps is 0."""
    from mimir_b200 import tensor as T
    x = matrix("random", (40, 72), 11) * factor
    check(x, T.orthogonalize(x, eps=0.0), eps=0.0)


def test_zeros_and_values_that_are_not_finite():
    from mimir_b200 import tensor as T
    x = matrix("random", (6, 40, 56), 12)
    want = T.orthogonalize(x)
    x[1] = 0
    x[2, 3, 4], x[3, 0, 0], x[5, 39, 55] = float("nan"), float("inf"), float("-inf")
    got = T.orthogonalize(x)
    assert not bool(got[1].any()) and bool(got[[2, 3, 5]].isnan().all()) and torch.equal(got[[0, 4]], want[[0, 4]])


def test_zeros_without_eps():
    from mimir_b200 import tensor as T
    for shape in ((40, 56), (200, 300), (130, 1)):
        assert not bool(T.orthogonalize(torch.zeros(shape, device="cuda"), eps=0.0).any())


def test_a_row_of_zeros_and_padding():
    from mimir_b200 import tensor as T
    x = matrix("random", (50, 80), 13)
    x[7], x[:, 11] = 0, 0
    got = T.orthogonalize(x)
    check(x, got)
    assert not bool(got[7].any()) and not bool(got[:, 11].any())


def test_same_bits_again_on_another_stream_and_in_a_graph():
    from mimir_b200 import tensor as T
    x = [matrix("random", (300, 520), 14), matrix("random", (3, 64, 48), 15)]
    want = T.orthogonalize(x)
    for _ in range(3):
        assert all(torch.equal(g, w) for g, w in zip(T.orthogonalize(x), want))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = T.orthogonalize(x)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = T.orthogonalize(x)
    before = x[0].clone()
    x[0].copy_(before.flip(0))
    graph.replay()
    assert torch.equal(got[0], T.orthogonalize(x[0])) and torch.equal(got[1], want[1])
    x[0].copy_(before)
    graph.replay()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_calls_on_several_streams_at_once():
    """Pairs of SMs and tensor memory asked for by several launches."""
    from mimir_b200 import tensor as T
    cases = [randn(shape, 40, 1.0, dtype) for shape, dtype in (((600, 900), F32), ((96, 64, 128), BF16), ((1500, 1100), BF16), ((40, 5000), F32))]
    want = [T.orthogonalize(x) for x in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(5):
        for stream, out, x in zip(streams, got, cases):
            with torch.cuda.stream(stream):
                out.append(T.orthogonalize(x))
    torch.cuda.synchronize()
    T.device_status()
    assert all(torch.equal(g, w) for out, w in zip(got, want) for g in out)


def test_refusals():
    import ctypes as C

    from mimir_b200 import MimkError, _lib
    from mimir_b200 import tensor as T
    x = matrix("random", (16, 24))
    with pytest.raises(ValueError, match="matrices"):
        T.orthogonalize(x[0])
    with pytest.raises(TypeError):
        T.orthogonalize(x.half())
    with pytest.raises(ValueError, match="CUDA tensors only"):
        T.orthogonalize([x, x.cpu()])
    for bad in (dict(steps=0), dict(coefficients=(1.0, 2.0)), dict(coefficients=((1.5, -0.5, 0.0),) * 4), dict(steps=2, coefficients=(1.5, -0.5, 0.0, 1.5, -0.5))):
        with pytest.raises(ValueError, match="three coefficients"):
            T.orthogonalize(x, **bad)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            T.orthogonalize(x, eps=eps)
    for bad in (dict(coefficients=(5.0, 0.0, 0.0)), dict(coefficients=(1.5, float("nan"), 0.0)), dict(steps=65)):
        with pytest.raises(MimkError) as e:
            T.orthogonalize(x, **bad)
        assert e.value.status == 8
    # the C entry point: addresses, and a workspace that is missing, too small or unaligned
    x = matrix("random", (16, 300))
    lib, need, out = _lib.lib(), C.c_uint64(), torch.empty((16, 300), dtype=BF16, device="cuda")
    d = _lib.OrthogonalizeDesc()
    d.batch, d.m, d.n, d.x, d.coefficients, d.eps, d.scale, d.steps, d.dtype = 1, 16, 300, (C.c_void_p * 1)(x.data_ptr()), (C.c_float * 3)(1.5, -0.5, 0.0), 1e-7, 1.0, 1, _lib.F32
    assert lib.mimk_orthogonalize_workspace(C.byref(d), C.byref(need)) == 0
    assert lib.mimk_orthogonalize(C.byref(d), None) == 1
    d.out = out.data_ptr()
    assert lib.mimk_orthogonalize(C.byref(d), None) == 9
    room = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = room.data_ptr(), need.value - 1
    assert lib.mimk_orthogonalize(C.byref(d), None) == 9
    d.workspace, d.workspace_bytes = room.data_ptr() + 4, need.value
    assert lib.mimk_orthogonalize(C.byref(d), None) == 3
    d.workspace, d.x = room.data_ptr(), (C.c_void_p * 1)(x.data_ptr() + 2)
    assert lib.mimk_orthogonalize(C.byref(d), None) == 3
    d.x = (C.c_void_p * 1)(None)
    assert lib.mimk_orthogonalize(C.byref(d), None) == 1
