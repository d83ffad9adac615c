"""The operators of a training step together, as the example of a model of tokens runs them: the gradients of all weights against automatic differentiation in 64 bits, the same
bits from a captured graph, and the example itself.

Tolerance of a gradient. Between the operators values are bf16, and within them h, da, db of a gated block and p of the cross-entropy are: each rounding is off by at most
2^-8 of its value. How such errors go on through the step the oracle finds: automatic differentiation in 64 bits with independent relative errors, uniform to that bound, on all of those values on the
way forward and on their gradients on the way back, eight times over. Positions of one token have the same values on the way forward, and so the same errors, which do not average out over them; on the
way back they differ by their targets only: positions of one token share their errors in a draw, both ways, which makes the sums' deviations no smaller than errors that are partly shared would. The roundings of
the step are one more such draw, of smaller errors (half a step's bound, three quarters of it on average over a binade, and none of the f32 weights'): a gradient's 2-norm error is allowed twice the
largest of the eight, and the rounding of the gradient itself."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PATH = os.path.join(ROOT, "examples", "train_tokens.py")
U = 2.0 ** -8


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_tokens", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class Off(torch.autograd.Function):
    """The value and its gradient, each off by a relative error of its own."""

    @staticmethod
    def forward(ctx, t, generator, ids, forward):
        ctx.generator, ctx.ids = generator, ids
        return t * error(t, generator, ids) if forward else t.clone()

    @staticmethod
    def backward(ctx, g):
        return g * error(g, ctx.generator, ctx.ids), None, None, None


def error(t, generator, ids):
    """1 and an error of each value; ids: positions, those of one id have the same."""
    if generator is None:
        return 1
    rows = t.shape[0] if ids is None else int(ids.max()) + 2
    e = 1 + U * (2 * torch.rand((rows, *t.shape[1:]), generator=generator, device=t.device, dtype=t.dtype) - 1)
    return e if ids is None else e[ids]


def oracle(w, ids, targets, seed=None):
    """(loss, {name: gradient}) in 64 bits."""
    generator = None if seed is None else torch.Generator(device="cuda").manual_seed(seed)
    off = lambda t, forward=True: Off.apply(t, generator, ids, forward)  # noqa: E731
    norm = lambda v, g: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * g  # noqa: E731
    p = {k: v.double().requires_grad_() for k, v in w.items()}
    there = (ids >= 0).unsqueeze(1)
    r = off(p["table"][ids.clamp(min=0)] * there * p["table"].shape[1] ** 0.5)
    x = off(norm(r, p["gamma"]))
    for i in range(sum(k.startswith("w1.") for k in w)):
        a, b = off(x @ p[f"w1.{i}"], False), off(x @ p[f"w3.{i}"], False)
        y = off(off(torch.nn.functional.silu(a) * b) @ p[f"w2.{i}"])
        r = off(r + p[f"gate.{i}"] * norm(y, p[f"post_gamma.{i}"]))
        x = off(norm(r, p[f"gamma.{i}"]))
    # (the table's two uses have a rounding of their gradient each)
    logits = off(x @ Off.apply(p["table"], generator, None, False).t(), False)
    loss = torch.nn.functional.cross_entropy(logits, targets, ignore_index=-1)
    return loss.detach(), dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def tokens(n, classes, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, classes, (n,), generator=g, device="cuda")
    targets = torch.randint(0, classes, (n,), generator=g, device="cuda")
    ids[3], targets[3], targets[n // 2], ids[: n // 4] = -1, -1, -1, 5       # no token, no target, a class of many positions
    return ids, targets


@pytest.mark.parametrize("n,classes,features,hidden,blocks", [(300, 500, 128, 320, 2), (3000, 301, 104, 200, 1), (64, 50, 33, 65, 3)])
def test_gradients_of_a_step(example, n, classes, features, hidden, blocks):
    w, (ids, targets) = example.weights(classes, features, hidden, blocks), tokens(n, classes, 1)
    loss, grads = example.gradients(w, ids, targets)
    want_loss, want = oracle(w, ids, targets)
    draws = [oracle(w, ids, targets, seed) for seed in range(8)]
    assert abs(float(loss) - float(want_loss)) <= 2 * max(abs(float(d[0] - want_loss)) for d in draws) + 1e-6 * abs(float(want_loss))
    assert grads.keys() == w.keys()
    for k, g in grads.items():
        assert g.shape == w[k].shape and g.dtype == w[k].dtype
        rounding = 1.01 * (U if g.dtype == torch.bfloat16 else 2.0 ** -24) * float(want[k].norm())
        allowed = 2 * max(float((d[1][k] - want[k]).norm()) for d in draws) + rounding
        assert float((g.double() - want[k]).norm()) <= allowed, k


def test_a_captured_step_beside_an_eager_one(example):
    """The same bits from a graph, replayed with other tokens, while another step runs on another stream."""
    w, (ids, targets) = example.weights(400, 96, 256, 2), tokens(2500, 400, 2)
    want = example.gradients(w, ids, targets)
    other_ids, other_targets = tokens(2500, 400, 3)
    other = example.gradients(w, other_ids, other_targets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = example.gradients(w, ids, targets)
    side = torch.cuda.Stream()
    for turn in range(4):
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            beside = example.gradients(w, other_ids, other_targets)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(loss, want[0]) and all(torch.equal(grads[k], want[1][k]) for k in grads)
        assert torch.equal(beside[0], other[0]) and all(torch.equal(beside[1][k], other[1][k]) for k in grads)
    ids.copy_(other_ids), targets.copy_(other_targets)
    graph.replay()
    assert torch.equal(loss, other[0]) and all(torch.equal(grads[k], other[1][k]) for k in grads)


def test_two_steps_on_two_streams(example):
    """Large enough that their launches overlap, those whose blocks meet among them."""
    from mimir_b200 import tensor as T
    n, classes, features = 20000, 30000, 512
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = [torch.randint(0, classes, (n,), generator=g, device="cuda") for _ in range(3)]
    dy = [torch.randn((n, features), generator=g, device="cuda").to(torch.bfloat16) for _ in range(3)]
    want = [T.embedding_grad(d, i, classes) for d, i in zip(dy, ids)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = [[] for _ in streams]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(T.embedding_grad(dy[k], ids[k], classes))
    torch.cuda.synchronize()
    T.device_status()
    assert all(torch.equal(t, want[k]) for k in range(3) for t in got[k])


def test_the_example_runs():
    r = subprocess.run([sys.executable, PATH, "--steps", "12"], capture_output=True, text=True, timeout=300, cwd="/")
    assert r.returncode == 0, r.stderr
    first, last = (float(v) for v in r.stdout.strip().splitlines()[-1].removeprefix("loss ").split(" -> "))
    assert first == first and last == last
