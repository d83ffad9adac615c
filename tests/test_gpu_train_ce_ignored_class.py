"""Cross-entropy of a linear layer whose ignored index is a class number (a padding token's, say), against the formulas in 64 bits: rows with that target
have none. Bounds are those of test_gpu_train_ce.py, from the formulas with such targets replaced by one that is no class.
"""
import pytest
import torch

from test_gpu_train_ce import BF16, E, F32, IGNORED, formulas, inputs, near

pytestmark = pytest.mark.gpu


def targets_with(t, ignore, share=0.4, seed=0):
    """t with about that share of the targets the ignored class, the first and the last of them among these; and the same as the formulas take it."""
    g = torch.Generator().manual_seed(seed)
    t = torch.where((torch.rand(t.shape, generator=g) < share).cuda(), torch.full_like(t, ignore), t)
    t[0] = t[-1] = ignore
    return t, torch.where(t == ignore, torch.full_like(t, IGNORED), t)


def classes(v):
    return sorted({0, v // 2, v - 1})


# one row (which is ignored); the pass of a few rows, of four and of fewer left; a tile and several; rows of no whole 16 bytes
SHAPES = [(1, 64, 1000), (2, 64, 500), (4, 136, 5001), (5, 128, 20000), (33, 72, 257), (300, 64, 513), (257, 5, 7)]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(shape, nk, dtype, index):
    from mimir_b200 import tensor as T
    x, w, t = inputs(*shape, dtype, nk)
    for ignore in classes(shape[2]):
        targets, known = targets_with(t, ignore)
        want, kept = formulas(x, w, known)
        bad = torch.where(kept[:, None], x, torch.full_like(x, float("nan")))          # what the ignored rows hold is not read
        targets = targets.to(index)
        losses, lse = T.linear_cross_entropy(bad, w, targets, ignore_index=ignore, reduction="none", return_lse=True)
        assert near(losses, *want[0]) and near(lse, *want[1])
        assert not bool(losses[~kept].any()) and not bool(lse[~kept].any())
        count = int(kept.sum())
        for reduction, over in (("mean", max(count, 1)), ("sum", 1)):
            total, bound = float(want[0][0].sum()) / over, float(want[0][1][kept].sum()) / over
            loss, dx, dw = T.linear_cross_entropy_with_grad(bad, w, targets, ignore_index=ignore, reduction=reduction)
            alone = T.linear_cross_entropy(bad, w, targets, ignore_index=ignore, reduction=reduction)
            for got in (loss, alone):
                assert abs(float(got) - total) <= bound + 1e-37 + E * abs(total)
            of_sum, _ = formulas(x, w, known, mean=reduction == "mean")
            assert near(dx, *of_sum[2]) and near(dw, *of_sum[3]) and not bool(dx[~kept].any())
            dx, dw = T.linear_cross_entropy_grad(bad, w, targets, lse, ignore_index=ignore, reduction=reduction)
            assert near(dx, *of_sum[2]) and near(dw, *of_sum[3]) and not bool(dx[~kept].any())
    T.device_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_that_arrive_at_each_loss(dtype):
    from mimir_b200 import tensor as T
    x, w, t = inputs(90, 48, 300, dtype, True)
    targets, known = targets_with(t, 0)
    g = torch.linspace(-1.0, 2.0, 90, device="cuda")
    want, kept = formulas(x, w, known, g.double(), mean=False)
    g = torch.where(kept, g, torch.full_like(g, float("nan")))                         # (nor is theirs)
    lse = T.linear_cross_entropy(x, w, targets, ignore_index=0, return_lse=True)[1]
    for dx, dw in (T.linear_cross_entropy_grad(x, w, targets, lse, ignore_index=0, reduction="none", dloss=g),
                   T.linear_cross_entropy_with_grad(x, w, targets, ignore_index=0, reduction="none", dloss=g)[1:]):
        assert near(dx, *want[2]) and near(dw, *want[3])
    T.device_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_class_is_ignored_only_where_it_is_asked_for(dtype):
    from mimir_b200 import tensor as T
    x, w, t = inputs(40, 64, 300, dtype, True, seed=2)
    t[:] = 0
    want, _ = formulas(x, w, t)
    assert near(T.linear_cross_entropy(x, w, t, reduction="none"), *want[0])
    assert near(T.linear_cross_entropy(x, w, t, ignore_index=299, reduction="none"), *want[0])
    loss, dx, dw = T.linear_cross_entropy_with_grad(x, w, t, ignore_index=0)
    assert float(loss) == 0 and not bool(dx.any()) and not bool(dw.any())
    T.device_status()


def test_an_index_of_more_than_64_bits():
    from mimir_b200 import tensor as T
    x, w, t = inputs(16, 32, 50, BF16, False)
    for index in (2 ** 64, 2 ** 63, -2 ** 63 - 1):          # (2^64 would be class 0 in the bits that are left)
        with pytest.raises(ValueError, match="64 bits"):
            T.linear_cross_entropy(x, w, t, ignore_index=index)
