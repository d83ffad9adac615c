"""The token embedding and its gradient against their definitions in 64 bits, through the public operators.

Tolerances. A result is rounded once to its type: half a step, u |result|, u = 2^-8 for bf16 and 2^-24 for f32. Before that there is one f32 product (2^-24 |result|), and for a
gradient the sum of c rows in f32: c - 1 additions, each off by at most 2^-24 of a partial sum, which is at most the sum of the magnitudes."""
import itertools

import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
E = 2.0 ** -24


def ids_of(shape, v, seed, dtype=torch.int64, skew=True):
    g = torch.Generator().manual_seed(seed)
    r = torch.rand(shape, generator=g, dtype=torch.float64)
    ids = ((v + 1) ** r - 1).long() if skew else (r * v).long()
    return ids.clamp(0, v - 1).to(dtype).cuda()


def check_forward(table, ids, scale, ignore, out_dtype):
    from mimir_b200 import tensor as T
    out = T.embedding(table, ids, scale=scale, ignore_index=ignore, out_dtype=out_dtype)
    T.device_status()
    assert out.dtype == (out_dtype or table.dtype) and tuple(out.shape) == (*ids.shape, table.shape[1])
    there = torch.ones_like(ids, dtype=torch.bool) if ignore is None else ids != ignore
    want = table.double()[torch.where(there, ids, 0).long()] * scale * there.unsqueeze(-1)
    assert bool(((out.double() - want).abs() <= (U[out.dtype] + E) * want.abs() * 1.01 + 1e-38).all())


def check_grad(dy, ids, v, scale, ignore, out_dtype=None, add_to=None):
    from mimir_b200 import tensor as T
    before = None if add_to is None else add_to.double()
    got = T.embedding_grad(dy, ids, v, scale=scale, ignore_index=ignore, out_dtype=out_dtype, add_to=add_to)
    T.device_status()
    d = dy.shape[-1]
    assert got.dtype == (add_to.dtype if add_to is not None else out_dtype or dy.dtype) and tuple(got.shape) == (v, d)
    there = (torch.ones_like(ids, dtype=torch.bool) if ignore is None else ids != ignore).reshape(-1)
    flat, rows = ids.reshape(-1).long()[there], dy.reshape(-1, d).double()[there]
    total = torch.zeros((v, d), dtype=torch.float64, device="cuda").index_add_(0, flat, rows) * scale
    size = torch.zeros((v, d), dtype=torch.float64, device="cuda").index_add_(0, flat, rows.abs()) * abs(scale)
    counts = torch.bincount(flat, minlength=v).double().unsqueeze(1)
    bound = (counts + 1) * E * size
    if before is not None:
        total, bound = total + before, bound + E * before.abs()
    bound = bound + U[got.dtype] * (total.abs() + bound)
    assert bool(((got.double() - total).abs() <= bound * 1.01 + 1e-38).all()), float(((got.double() - total).abs() / (bound + 1e-38)).max())
    none = (counts == 0).squeeze(1)
    if before is None:
        assert not bool(got[none].any())
    else:
        assert torch.equal(got[none].double(), before[none])
    return got


# one value; fewer columns than a warp, rows of no whole 16 bytes; a part's columns, and past them; more positions than classes
SHAPES = [(1, 1, 1), (3, 7, 5), (33, 31, 2), (64, 512, 40), (65, 520, 1000), (1000, 72, 300), (2000, 1032, 77), (257, 255, 10007), (5000, 64, 3)]


@pytest.mark.parametrize("shape,dtype", list(itertools.product(SHAPES, [BF16, F32])))
def test_forward_and_gradient(shape, dtype):
    n, d, v = shape
    ids = ids_of((n,), v, n, torch.int32 if n % 2 else torch.int64)
    check_forward(randn((v, d), 1, 1.0, dtype), ids, 1.0, None, None)
    check_forward(randn((v, d), 1, 1.0, dtype), ids, 22.625, 0, F32 if dtype == BF16 else BF16)
    dy = randn((n, d), 2, 1.0, dtype)
    check_grad(dy, ids, v, 1.0, None)
    check_grad(dy, ids, v, -0.375, 0, F32 if dtype == BF16 else BF16)


@pytest.mark.parametrize("count", [1, 2, 31, 32, 33, 64, 255, 256, 257, 1000, 2047, 2048, 2049, 4096, 9000])
def test_runs_of_one_class(count):
    """Classes of every number of positions around where another way of adding them up is taken, others among them."""
    d, v = 136, 50
    ids = torch.full((count + 40,), 17, dtype=torch.int64)
    ids[torch.randperm(count + 40, generator=torch.Generator().manual_seed(count))[:40]] = torch.arange(40) % 11 + 20
    check_grad(randn((count + 40, d), 3, 1.0, BF16), ids.cuda(), v, 1.0, None, F32)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_table(dtype):
    ids = ids_of((2, 3000), 50021, 5)
    check_forward(randn((50021, 264), 1, 1.0, dtype), ids, 3.0, None, None)
    check_grad(randn((2, 3000, 264), 2, 1.0, dtype), ids, 50021, 1.0, None)


def test_many_positions():
    """More positions than one map of bits holds, a class that half of them name."""
    n = 300001
    ids = ids_of((n,), 40, 6)
    ids[::2] = 7
    check_grad(randn((n, 24), 2, 1.0, BF16), ids, 40, 1.0, None, F32)


def test_many_classes_of_many_positions():
    """More positions than one map of bits holds: classes of some hundred, of a few thousand, of more than are sorted in shared memory, and of more than a map's."""
    from mimir_b200 import tensor as T
    n, v = 400001, 1000
    ids = ids_of((n,), v, 7, skew=False)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(7)).cuda()
    ids[order[:4000]], ids[order[4000:8500]], ids[order[8500:150000]] = 3, 500, v - 1
    dy = randn((n, 16), 2, 1.0, F32)
    assert torch.equal(check_grad(dy, ids, v, 1.0, None), T.embedding_grad(dy, ids, v))


def test_one_class_of_very_many_positions():
    """Whole numbers, so that sums are exact in whichever order."""
    from mimir_b200 import tensor as T
    n, v = 2 ** 25 + 3, 4
    ids = torch.full((n,), 2, dtype=torch.int32, device="cuda")
    ids[::1001] = 1
    dy = torch.randint(-1, 2, (n, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).float()
    got = T.embedding_grad(dy, ids, v)
    T.device_status()
    assert torch.equal(got[:, 0], torch.stack([dy[ids == c].double().sum() for c in range(v)]).float())


def test_add_to():
    from mimir_b200 import tensor as T
    for n, d, v in ((700, 264, 200), (700, 33, 5000), (10, 64, 90)):
        for dtype, kept in ((BF16, BF16), (BF16, F32), (F32, F32)):
            ids, dy = ids_of((n,), v, 8), randn((n, d), 9, 1.0, dtype)
            room = randn((v, d), 10, 1.0, kept)
            version = room._version
            assert check_grad(dy, ids, v, 0.75, 3, add_to=room) is room and room._version > version
    # rows that no position names keep even what is not finite
    room = torch.full((50, 16), float("nan"), dtype=BF16, device="cuda")
    room[4] = 1.0
    T.embedding_grad(torch.ones((2, 16), dtype=BF16, device="cuda"), torch.tensor([4, 4], device="cuda"), 50, add_to=room)
    assert bool((room[4] == 3.0).all()) and int(room.isnan().sum()) == 49 * 16


def test_ignored_positions_are_not_read():
    from mimir_b200 import tensor as T
    ids = ids_of((400,), 60, 11)
    ids[::3] = -1
    dy = randn((400, 40), 12, 1.0, BF16)
    want = T.embedding_grad(dy, ids, 60, ignore_index=-1)
    dy[::3] = float("nan")
    assert torch.equal(T.embedding_grad(dy, ids, 60, ignore_index=-1), want)
    out = T.embedding(randn((60, 40), 13, 1.0, F32), ids, ignore_index=-1)
    assert not bool(out[::3].any())
    # all of them ignored, and an ignored index that is a class
    assert not bool(T.embedding_grad(dy, torch.full_like(ids, -1), 60, ignore_index=-1).any())
    assert not bool(T.embedding(randn((60, 40), 13, 1.0, F32), torch.full_like(ids, 5), ignore_index=5).any())


@pytest.mark.parametrize("bad", [-1, 60, 2 ** 31, -2 ** 40, 2 ** 63 - 1])
def test_ids_that_are_no_class(bad):
    from mimir_b200 import MimkError
    from mimir_b200 import tensor as T
    ids = ids_of((90,), 60, 14)
    table, dy = randn((60, 40), 13, 1.0, BF16), randn((90, 40), 12, 1.0, BF16)
    wrong = ids.clone()
    wrong[[5, 44, 45]] = bad
    out = T.embedding(table, wrong)
    with pytest.raises(MimkError):
        T.device_status()
    keep = torch.ones(90, dtype=torch.bool, device="cuda")
    keep[[5, 44, 45]] = False
    assert bool(out[~keep].isnan().all()) and torch.equal(out[keep], T.embedding(table, ids)[keep])
    T.device_status()
    grad = T.embedding_grad(dy, wrong, 60)
    with pytest.raises(MimkError):
        T.device_status()
    assert torch.equal(grad, T.embedding_grad(dy[keep], ids[keep], 60))
    T.device_status()


def test_infinities_and_nan_stay_in_their_classes():
    from mimir_b200 import tensor as T
    ids, dy = ids_of((300,), 30, 15, skew=False), randn((300, 48), 16, 1.0, BF16)
    want = T.embedding_grad(dy, ids, 30)
    dy[7, 3], dy[8, 5] = float("nan"), float("inf")
    got = T.embedding_grad(dy, ids, 30)
    assert bool(got[ids[7], 3].isnan()) and bool(got[ids[8], 5].isinf())
    got[ids[7], 3], got[ids[8], 5] = want[ids[7], 3], want[ids[8], 5]
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,d,v", [(0, 16, 9), (5, 0, 9), (0, 0, 0), (0, 16, 0)])
def test_empty_extents(n, d, v):
    from mimir_b200 import tensor as T
    ids = torch.zeros((n,), dtype=torch.int64, device="cuda")
    assert tuple(T.embedding(randn((v, d), 1, 1.0, F32), ids).shape) == (n, d)
    g = T.embedding_grad(randn((n, d), 1, 1.0, F32), ids, v)
    assert tuple(g.shape) == (v, d) and not bool(g.any())
    T.device_status()


def test_no_classes():
    from mimir_b200 import MimkError
    from mimir_b200 import tensor as T
    assert bool(T.embedding(randn((0, 8), 1, 1.0, F32), torch.zeros((3,), dtype=torch.int64, device="cuda")).isnan().all())
    with pytest.raises(MimkError):
        T.device_status()


def test_shapes_strides_and_addresses():
    from mimir_b200 import tensor as T
    ids, table, dy = ids_of((4, 5, 6), 70, 17), randn((70, 64), 18, 1.0, BF16), randn((4, 5, 6, 64), 19, 1.0, BF16)
    out, grad = T.embedding(table, ids), T.embedding_grad(dy, ids, 70)
    assert torch.equal(T.embedding(table, ids[2, 3, 4]), table[ids[2, 3, 4]]) and tuple(T.embedding(table, ids[2, 3, 4]).shape) == (64,)

    def moved(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:].copy_(t.reshape(-1))
        return room[1:].view(t.shape)

    def wide(t):
        room = torch.full((*t.shape[:-1], t.shape[-1] + 3), 1, dtype=t.dtype, device="cuda")
        room[..., :t.shape[-1]] = t
        return room[..., :t.shape[-1]]

    for change in (moved, wide, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(T.embedding(change(table), change(ids)), out)
        assert torch.equal(T.embedding_grad(change(dy), change(ids), 70), grad)
    # (a result elsewhere than on 16 bytes is added to in the same order)
    room = torch.zeros(70 * 64 + 1, dtype=BF16, device="cuda")[1:].view(70, 64)
    assert torch.equal(T.embedding_grad(dy, ids, 70, add_to=room), grad)


def test_rows_that_begin_past_32_bits():
    """A table of more than 2^32 bytes and 2^31 elements, its last rows among the tokens."""
    from mimir_b200 import tensor as T
    v, d = 2 ** 31 // 4096 + 64, 4096
    table = torch.zeros((v, d), dtype=BF16, device="cuda")
    table[-8:] = randn((8, d), 20, 1.0, BF16)
    ids = torch.tensor([v - 1, 0, v - 8, v - 1], device="cuda")
    assert torch.equal(T.embedding(table, ids), table[ids])
    dy = randn((4, d), 21, 1.0, BF16)
    table.zero_()
    T.embedding_grad(dy, ids, v, add_to=table)
    assert torch.equal(table[v - 8], dy[2]) and torch.equal(table[0], dy[1])
    assert torch.equal(table[v - 1], (dy[0].float() + dy[3].float()).to(BF16)) and int(table.any(1).sum()) == 3


def test_same_bits_again_on_another_stream_and_in_a_graph():
    from mimir_b200 import tensor as T
    ids, table, dy = ids_of((5000,), 800, 22), randn((800, 264), 23, 1.0, BF16), randn((5000, 264), 24, 1.0, BF16)
    run = lambda: (T.embedding(table, ids, scale=3.0), T.embedding_grad(dy, ids, 800, scale=3.0, out_dtype=F32))  # noqa: E731
    want = run()
    for _ in range(3):
        assert all(torch.equal(g, w) for g, w in zip(run(), want))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = run()
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    ids_before = ids.clone()
    for turn in range(2):      # other ids in the same graph
        ids.copy_(ids_before if turn else ids_before.flip(0))
        graph.replay()
        assert all(torch.equal(g, w) for g, w in zip(got, run()))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_calls_on_several_streams_at_once():
    """Launches whose blocks meet, beside one another and beside products that fill the GPU."""
    from mimir_b200 import tensor as T
    cases = [(randn((n, 512), n, 1.0, BF16), ids_of((n,), v, n), v) for n, v in ((5000, 20011), (8192, 300), (2500, 50021), (1000, 4000))]
    want = [T.embedding_grad(dy, ids, v) for dy, ids, v in cases]
    a = randn((4096, 4096), 1, 1.0, BF16)
    product = T.product_2d(a, a)
    streams = [torch.cuda.Stream() for _ in range(len(cases) + 1)]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(6):
        with torch.cuda.stream(streams[-1]):
            same = T.product_2d(a, a)
        for stream, out, (dy, ids, v) in zip(streams, got, cases):
            with torch.cuda.stream(stream):
                out.append(T.embedding_grad(dy, ids, v))
    torch.cuda.synchronize()
    T.device_status()
    assert torch.equal(same, product) and all(torch.equal(g, w) for out, w in zip(got, want) for g in out)


def test_gradient_against_differences():
    """<out, dy> along a step of the table: the forward pass is linear, so the quotient is the product with the gradient but for the roundings of both."""
    from mimir_b200 import tensor as T
    ids, table, dy = ids_of((300,), 50, 25), randn((50, 40), 26, 1.0, F32), randn((300, 40), 27, 1.0, F32)
    grad = T.embedding_grad(dy, ids, 50, scale=1.75).double()
    step = torch.sign(grad).float()
    plus, minus = table + step, table - step
    quotient = float(((T.embedding(plus, ids, scale=1.75).double() - T.embedding(minus, ids, scale=1.75).double()) * dy.double()).sum())
    slope = float((grad * (plus.double() - minus.double())).sum())
    allowed = 2 * E * float((T.embedding(plus.abs().maximum(minus.abs()), ids, scale=1.75).double() * dy.double().abs()).sum()) + 303 * E * 2 * float(
        T.embedding_grad(dy.abs(), ids, 50, scale=1.75).double().sum())
    assert abs(quotient - slope) <= allowed and slope > 100 * allowed


def test_refusals():
    import ctypes as C

    from mimir_b200 import _lib
    from mimir_b200 import tensor as T
    ids, table, dy = ids_of((20,), 50, 28), randn((50, 40), 29, 1.0, BF16), randn((20, 40), 30, 1.0, BF16)
    with pytest.raises(ValueError, match="rank 2"):
        T.embedding(table[0], ids)
    for bad in (ids.float(), ids.to(torch.int16)):
        with pytest.raises(TypeError, match="ids"):
            T.embedding(table, bad)
    with pytest.raises(TypeError):
        T.embedding(table.half(), ids)
    with pytest.raises(TypeError):
        T.embedding(table, ids, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="64 bits"):
        T.embedding(table, ids, ignore_index=2 ** 63)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        T.embedding(table.cpu(), ids)
    with pytest.raises(ValueError, match="one row of dy"):
        T.embedding_grad(dy[:19], ids, 50)
    with pytest.raises(ValueError, match="at least 0"):
        T.embedding_grad(dy, ids, -1)
    for bad in (table[:49], table.t().contiguous().t(), randn((50, 41), 1)[:, :40]):
        with pytest.raises(ValueError, match="add_to"):
            T.embedding_grad(dy, ids, 50, add_to=bad)
    with pytest.raises(TypeError):
        T.embedding_grad(dy, ids, 50, add_to=table, out_dtype=F32)
    # the C entry points: addresses, and a workspace that is missing, too small or unaligned
    lib, need = _lib.lib(), C.c_uint64()
    d = _lib.EmbeddingDesc()
    out = torch.empty_like(table)
    ids, dy = ids_of((3000,), 50, 28), randn((3000, 40), 30, 1.0, BF16)
    d.n, d.d, d.v, d.ids, d.dy, d.scale, d.dtype, d.out_dtype, d.id_dtype = 3000, 40, 50, ids.data_ptr(), dy.data_ptr(), 1.0, _lib.BF16, _lib.BF16, _lib.I64
    assert lib.mimk_embedding_grad(C.byref(d), None) == 1
    d.dtable = out.data_ptr()
    assert lib.mimk_embedding_grad_workspace(C.byref(d), C.byref(need)) == 0
    assert lib.mimk_embedding_grad(C.byref(d), None) == 9
    room = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = room.data_ptr(), need.value - 1
    assert lib.mimk_embedding_grad(C.byref(d), None) == 9
    d.workspace, d.workspace_bytes = room.data_ptr() + 4, need.value
    assert lib.mimk_embedding_grad(C.byref(d), None) == 3
    d.workspace, d.dy = room.data_ptr(), dy.data_ptr() + 1
    assert lib.mimk_embedding_grad(C.byref(d), None) == 3
    assert lib.mimk_embedding(C.byref(d), None) == 1
