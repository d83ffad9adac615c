"""linear_cross_entropy_grad takes each row's log sum exp from its caller: gradients with p = exp(l - lse) for whatever lse is given, both element types
alike. Tolerances as in test_gpu_train_ce.py, which p = exp(l - lse) of an exact lse only makes smaller."""
import pytest
import torch

from test_gpu_train_ce import BF16, E, F32, IGNORED, U, inputs, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("shape", [(1, 64, 1000), (5, 33, 70), (130, 72, 1031)])
def test_the_given_lse_counts(shape, nk, dtype):
    from mimir_b200 import tensor as T
    n, d, v = shape
    x, w, t = inputs(*shape, dtype, nk, masked=0.3)
    t[0] = 1
    kept = t >= 0
    of_call = T.linear_cross_entropy(x, w, t, ignore_index=IGNORED, reduction="none", return_lse=True)[1]
    terms = 0 if dtype == BF16 else 2.0 ** -20
    x64, w64 = torch.where(kept[:, None], x.double(), 0.0), w.double()
    l = x64 @ w64
    el = x64.abs() @ w64.abs() * (d * E / 2 + terms)
    one = torch.zeros_like(l).scatter_(1, torch.where(kept, t, 0)[:, None], 1.0)
    for shift in (0.0, 1.5, -0.25):
        # (a softmax over a part of the classes, or over more than there are here, has another sum)
        lse = torch.where(kept, of_call + shift, float("nan"))
        at = lse.double()[:, None].nan_to_num(0.0)
        p = torch.exp(l - at)
        dl = kept[:, None] * (p - one)
        edl = kept[:, None] * (p * (el * 1.01 + E * (8 + (l - at).abs() + at.abs())) + E * one) + (4 * E + (U if dtype == BF16 else 0)) * dl.abs()
        want = []
        for left, right, eleft, eright, k in ((dl, w64.t(), edl, w64.t().abs(), v), (x64.t(), dl, x64.t().abs(), edl, n)):
            exact = left @ right
            want.append((exact, 1.02 * (eleft @ eright + (k * E + terms) * (left.abs() @ right.abs()) + (U if dtype == BF16 else E) * exact.abs()) + 1e-37))
        got = T.linear_cross_entropy_grad(x, w, t, lse, ignore_index=IGNORED, reduction="sum")
        assert near(got[0], *want[0]) and near(got[1], *want[1]), shift
    T.device_status()


def test_no_lse():
    from mimir_b200 import tensor as T
    x, w, t = inputs(16, 32, 50, F32, False)
    with pytest.raises(ValueError, match="lse"):
        T.linear_cross_entropy_grad(x, w, t, None)
