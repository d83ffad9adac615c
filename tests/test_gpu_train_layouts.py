"""Training operators whose matrices have an axis of one value: such a matrix is row-major and a transposed view of a row-major one at once, and its strides
along that axis mean nothing."""
import pytest
import torch

from test_gpu_train_mlp import formulas, inputs, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("one", range(4))
def test_gated_mlp(one, nk):
    shape = [40, 72, 136, 48]
    shape[one] = 1
    args = inputs(*shape, nk, seed=1)
    for g, (want, bound) in zip(step(*args), formulas(*args)):
        assert g.shape == want.shape and bool(((g.double() - want).abs() <= bound).all())


def test_gated_mlp_with_one_weight_that_is_copied():
    args = list(inputs(40, 72, 136, 48, True, seed=2))
    want = step(*args)
    wide = torch.zeros((72, 2 * 136), dtype=args[1].dtype, device="cuda")
    wide[:, ::2] = args[1]
    args[1] = wide[:, ::2]                                  # neither layout; the others are transposed views
    for g, w in zip(step(*args), want):
        assert torch.equal(g, w)
