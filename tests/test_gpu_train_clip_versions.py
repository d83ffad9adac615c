"""clip_grad_norm changes tensors in place: their version counters say so, and autograd refuses a backward pass through values that it saved before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class _General:
    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture(params=["native", "general"])
def T(request, monkeypatch):
    from mimir_b200 import tensor
    if request.param == "general":
        monkeypatch.setattr(tensor, "_native", _General())
    return tensor


@pytest.mark.parametrize("limit", [1e-3, 1e6])
def test_version_counters(T, limit):
    a, b, view = torch.randn(1000, device="cuda"), torch.randn(3, 5, device="cuda").bfloat16(), torch.randn(64, device="cuda")[16:48]
    out = [torch.empty_like(t) for t in (a, b, view)]
    before = [t._version for t in (a, b, view._base, *out)]
    T.grad_norm([a, b, view])
    T.clip_grad_norm([a, b, view], limit, out=out)
    assert [t._version for t in (a, b, view._base)] == before[:3]
    assert all(t._version > v for t, v in zip(out, before[3:]))
    T.clip_grad_norm([a, b, view], limit)
    assert all(t._version > v for t, v in zip((a, b, view._base), before))


def test_a_saved_gradient_that_was_clipped(T):
    x = torch.randn(50, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    twice = (g * g).sum()                                    # (saves g)
    T.clip_grad_norm([g.detach()], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        twice.backward()


def test_inference_tensors(T):
    with torch.inference_mode():
        g = torch.ones(40, device="cuda")
        T.clip_grad_norm([g], 1.0)
    T.clip_grad_norm([g], 0.5)
    assert abs(float(g.double().norm()) - 0.5) < 1e-6
