"""clip_grad_norm into results whose strides differ from the gradients' only where they mean nothing: along axes of one value, or of a tensor without values."""
import pytest
import torch

from test_gpu_train_clip import holds, reference
from util import randn

pytestmark = pytest.mark.gpu


def test_strides_that_mean_nothing():
    from mimir_b200 import tensor as T
    grads = [randn((50, 1), 1).t(), randn((7, 1, 9), 2).transpose(0, 1), torch.empty((0, 6), device="cuda").t(), randn((4, 6), 3).t()]
    out = [torch.empty((1, 50), device="cuda"), torch.empty((1, 7, 9), device="cuda"), torch.empty((6, 0), device="cuda"), torch.empty((4, 6), device="cuda").t()]
    assert any(g.stride() != o.stride() for g, o in zip(grads, out))
    for some in (range(4), (0, 1, 3)):
        ins, outs = [grads[i] for i in some], [out[i] for i in some]
        want_norm, want = reference(ins, 1.0)
        holds(T.clip_grad_norm(ins, 1.0, out=outs), outs, want_norm, want)
    for bad in (torch.empty((6, 4), device="cuda"), torch.empty((6, 8), device="cuda")[:, ::2]):
        with pytest.raises(ValueError, match="same shape and strides"):
            T.clip_grad_norm([grads[3]], 1.0, out=[bad])
