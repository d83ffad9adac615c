"""A training step of one transformer-like block, gradients and all: a gated MLP with a residual connection under a linear output layer.

    python examples/train_block.py [--steps N]

Rows of features get class numbers from a hidden linear teacher; some rows have none. Each step is forward (mlp_gated_fwd, binary add), loss with
gradients (linear_cross_entropy_with_grad), backward (mlp_gated_bwd), clipping (clip_grad_norm) and plain gradient descent. Prints the loss
and the gradients' norm as it goes.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mimir_b200 import tensor as T  # noqa: E402

IGNORED = -100


def train(steps: int, rows: int = 512, features: int = 256, hidden: int = 704, classes: int = 1000, rate: float = 2.0, limit: float = 0.1, seed: int = 0):
    """The losses of `steps` steps."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, std=1.0: (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)  # noqa: E731
    x = normal(rows, features)
    targets = T.product_2d(x, normal(features, classes), out_dtype=torch.float32).argmax(1)
    targets[::7] = IGNORED
    weights = [normal(features, hidden, std=features ** -0.5), normal(features, hidden, std=features ** -0.5), normal(hidden, features, std=hidden ** -0.5),
               normal(classes, features, std=features ** -0.5)]
    losses = []
    for step in range(steps):
        w1, w3, w2, head = weights
        y, kept = T.mlp_gated_fwd(x, w1, w3, w2)
        loss, dy, dhead = T.linear_cross_entropy_with_grad(T.binary("add", x, y), T.transpose_2d(head), targets, ignore_index=IGNORED)
        _, dw1, dw3, dw2 = T.mlp_gated_bwd(dy, x, w1, w3, w2, kept)
        grads = [dw1, dw3, dw2, T.transpose_2d(dhead)]
        norm = T.clip_grad_norm(grads, limit)
        for w, d in zip(weights, grads):
            w.sub_(d, alpha=rate)
        losses.append(float(loss))
        if step % 10 == 0:
            print(f"step {step:4d}  loss {losses[-1]:.4f}  gradient norm {float(norm):.4f}", flush=True)
    T.device_status()
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=60)
    losses = train(parser.parse_args().steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
