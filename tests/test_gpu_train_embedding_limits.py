"""The embedding's gradient at the ends of its ranges. Values are small whole numbers, so that sums in f32 are exact: every row has to be equal."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def test_as_many_classes_as_there_can_be():
    """2^31 - 1 classes of one feature, of few positions: the last ones are written as the first, and no row is left as it was."""
    from mimir_b200 import _lib
    from mimir_b200 import tensor as T
    v = 2 ** 31 - 1
    for id_dtype, code in ((torch.int32, _lib.I32), (torch.int64, _lib.I64)):
        ids = torch.tensor([0, v - 1, 1, v - 2, 1 << 30, v - 1, v - 1024, 1023], dtype=id_dtype, device="cuda")
        dy = torch.arange(1, 9, device="cuda", dtype=F32).to(BF16).view(8, 1)
        out = torch.full((v, 1), float("nan"), dtype=BF16, device="cuda")
        d = _lib.EmbeddingDesc()
        d.n, d.d, d.v, d.ids, d.dy, d.dtable, d.scale = 8, 1, v, ids.data_ptr(), dy.data_ptr(), out.data_ptr(), 1.0
        d.dtype, d.out_dtype, d.id_dtype = _lib.BF16, _lib.BF16, code
        assert _lib.lib().mimk_embedding_grad(C.byref(d), torch.cuda.current_stream().cuda_stream) == 0
        there = {0: 1, 1: 3, 1023: 8, 1 << 30: 5, v - 1024: 7, v - 2: 4, v - 1: 2 + 6}
        assert all(float(out[c]) == w for c, w in there.items())
        for c in there:
            out[c] = 0
        assert not any(bool(part.ne(0).any()) for part in out.split(1 << 28))
        del out
    T.device_status()


@pytest.mark.parametrize("classes, each", [(148, 151552), (300, 37888), (37, 200000), (2000, 300), (1000, 40)])
def test_classes_whose_pieces_are_a_multiple_of_the_blocks(classes, each):
    """Groups of as many pieces as there are blocks, or a multiple: putting them in order is no one block's work. Positions of all classes in turn, and a class of few positions after each."""
    from mimir_b200 import tensor as T
    ids = torch.arange(classes, device="cuda", dtype=torch.int32).repeat(each) * 2
    ids = torch.cat([ids, torch.arange(classes, device="cuda", dtype=torch.int32).repeat(3) * 2 + 1])
    dy = torch.ones((ids.numel(), 1), device="cuda", dtype=BF16)
    for _ in range(2):
        got = T.embedding_grad(dy, ids, 2 * classes, out_dtype=F32).view(classes, 2)
        T.device_status()
        assert bool((got[:, 0] == each).all()) and bool((got[:, 1] == 3).all())


def test_order_of_sums_where_many_classes_have_many_positions():
    """Sums in f32 that depend on their order (magnitudes from 1 to 2^20): in groups of 512 positions and of a warp's share of those, in rising order, whichever block put the group in order."""
    from mimir_b200 import tensor as T
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(0, 700, (1 << 20,), generator=g, device="cuda")
    dy = torch.randn((1 << 20, 8), generator=g, device="cuda") * torch.exp2(torch.randint(0, 21, (1 << 20, 1), generator=g, device="cuda").float())
    want = T.embedding_grad(dy, ids, 700)
    assert all(torch.equal(T.embedding_grad(dy, ids, 700), want) for _ in range(5))
    exact = torch.zeros((700, 8), dtype=torch.float64, device="cuda").index_add_(0, ids, dy.double())
    sums = torch.zeros((700, 8), dtype=torch.float64, device="cuda").index_add_(0, ids, dy.double().abs())
    # 1500 or so positions of a class: no more than 32 of a warp's, 16 warps' and 4 pieces' sums one after another, each off by half a step of the magnitudes' sum at most
    assert bool(((want.double() - exact).abs() <= (32 + 16 + 4 + 1) * 2.0 ** -24 * sums).all())
    T.device_status()
