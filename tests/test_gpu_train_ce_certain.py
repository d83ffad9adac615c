"""Gradients of the cross-entropy for rows that are nearly certain of their target: softmax - 1 there is the difference of a logit and the lse that it went
into, and says nothing if the two were rounded in different ways.

Tolerance. With l and lse of the same rounded logits, softmax - 1 moves by |softmax - 1| times twice a logit's error e_l (as in test_gpu_train_ce.py), and by the
roundings of lse (8 + |lse| units of 2^-22), of l - lse and of exp (8 more). In bf16 it is rounded, and the gradient again."""
import pytest
import torch

from test_gpu_train_ce import BF16, E, F32, U
from util import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("d", [64, 1024, 1088, 4096])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 64])
def test_rows_that_are_nearly_certain(n, d, nk, dtype):
    from mimir_b200 import tensor as T
    v = 1000
    w = randn((v, d), d, d ** -0.5, F32)
    t = (torch.arange(n, device="cuda") * 37 + 11) % v
    x = w[t] * torch.linspace(15.0, 30.0, n, device="cuda")[:, None] / (w[t] ** 2).sum(1, keepdim=True)
    x, w = x.to(dtype), w.to(dtype).t()
    w = w if nk else w.contiguous()
    l = x.double() @ w.double()
    true = (torch.softmax(l, 1) - 1).gather(1, t[:, None])[:, 0]
    el = (x.double().abs() @ w.double().abs()).max(1).values * (d * E / 2 + (0 if dtype == BF16 else 2.0 ** -20))
    round_off = 2.1 * U if dtype == BF16 else 4 * E + 2.0 ** -20
    bound = true.abs() * (round_off + 2 * el) + E * (24 + 2 * torch.logsumexp(l, 1).abs())
    lse = T.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)[1]
    for i in sorted({0, n // 2, n - 1}):
        only = torch.zeros(n, device="cuda")
        only[i] = 1                                          # the gradient of this row's loss: dw of its target's column is (softmax - 1) x
        for name, (dx, dw) in (("from lse", T.linear_cross_entropy_grad(x, w, t, lse, reduction="none", dloss=only)),
                               ("at once", T.linear_cross_entropy_with_grad(x, w, t, reduction="none", dloss=only)[1:])):
            row = x[i].double()
            got = float((dw[:, t[i]].double() * row).sum() / (row * row).sum())
            assert abs(got - float(true[i])) <= float(bound[i]), (name, i, got, float(true[i]))
    T.device_status()
