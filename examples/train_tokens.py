"""A training step of a small model of tokens, from the ids to the updated weights: embedding, blocks of a gated MLP between two norms and a learned gate each, and an output
layer that shares the embedding's table.

    python examples/train_tokens.py [--steps N]

Tokens follow a hidden table of successors; the model learns the next one from each. A step is forward (embedding, residual_rmsnorm_fwd, mlp_gated_fwd), loss with gradients
(linear_cross_entropy_with_grad), backward (residual_rmsnorm_bwd, mlp_gated_bwd, embedding_grad, which adds to the output layer's gradient of the shared table), clipping
(clip_grad_norm) and the update: the momentum of the weight matrices made orthogonal (orthogonalize), plain gradient descent for the rest.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mimir_b200 import tensor as T  # noqa: E402

NO_TOKEN, EPS = -1, 1e-6


def weights(classes: int, features: int, hidden: int, blocks: int, seed: int = 0):
    """{name: tensor}: the table, the first norm's weights, and each block's."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, std: (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)  # noqa: E731
    w = dict(table=normal(classes, features, std=features ** -0.5), gamma=torch.ones(features, device="cuda"))
    for i in range(blocks):
        w.update({f"w1.{i}": normal(features, hidden, std=features ** -0.5), f"w3.{i}": normal(features, hidden, std=features ** -0.5),
                  f"w2.{i}": normal(hidden, features, std=hidden ** -0.5), f"post_gamma.{i}": torch.ones(features, device="cuda"),
                  f"gate.{i}": torch.full((features,), 0.5, device="cuda"), f"gamma.{i}": torch.ones(features, device="cuda")})
    return w


def gradients(w, ids: torch.Tensor, targets: torch.Tensor):
    """The loss of the tokens `ids` against the tokens that follow, and {name: gradient}; positions whose id or target is NO_TOKEN have none."""
    classes, features = w["table"].shape
    blocks, scale = sum(name.startswith("w1.") for name in w), float(features) ** 0.5
    r = T.embedding(w["table"], ids, scale=scale, ignore_index=NO_TOKEN)
    r, x, kept = T.residual_rmsnorm_fwd(r, None, w["gamma"], EPS)
    first, passed = (r, kept), []
    for i in range(blocks):
        y, mlp = T.mlp_gated_fwd(x, w[f"w1.{i}"], w[f"w3.{i}"], w[f"w2.{i}"])
        more = dict(post_gamma=w[f"post_gamma.{i}"], gate=w[f"gate.{i}"])
        new, out, kept = T.residual_rmsnorm_fwd(r, y, w[f"gamma.{i}"], EPS, **more)
        passed.append((x, mlp, r, y, kept, more))
        r, x = new, out
    loss, dx, dhead = T.linear_cross_entropy_with_grad(x, T.transpose_2d(w["table"]), targets, ignore_index=NO_TOKEN)
    grads, dr = {}, None
    for i in reversed(range(blocks)):
        x, mlp, r, y, kept, more = passed[i]
        dr, dy, grads[f"gamma.{i}"], grads[f"post_gamma.{i}"], grads[f"gate.{i}"] = T.residual_rmsnorm_bwd(dr, dx, r, y, w[f"gamma.{i}"], kept, **more)
        dx, grads[f"w1.{i}"], grads[f"w3.{i}"], grads[f"w2.{i}"] = T.mlp_gated_bwd(dy, x, w[f"w1.{i}"], w[f"w3.{i}"], w[f"w2.{i}"], mlp)
    dr, _, grads["gamma"], _, _ = T.residual_rmsnorm_bwd(dr, dx, first[0], None, w["gamma"], first[1])
    grads["table"] = T.embedding_grad(dr, ids, classes, scale=scale, ignore_index=NO_TOKEN, add_to=T.transpose_2d(dhead))
    return loss, grads


def train(steps: int, tokens: int = 1024, classes: int = 1000, features: int = 256, hidden: int = 704, blocks: int = 2, rate: float = 0.02, limit: float = 1.0, seed: int = 0):
    """The losses of `steps` steps."""
    w = weights(classes, features, hidden, blocks, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    follows = torch.randperm(classes, generator=g, device="cuda")
    matrices = [name for name in w if w[name].dim() == 2 and name != "table"]
    momentum = {name: torch.zeros_like(w[name], dtype=torch.float32) for name in matrices}
    losses = []
    for step in range(steps):
        ids = torch.randint(0, classes, (tokens,), generator=g, device="cuda")
        targets = follows[ids]
        ids[-7:] = NO_TOKEN             # the batch's padding
        targets[-7:] = NO_TOKEN
        loss, grads = gradients(w, ids, targets)
        norm = T.clip_grad_norm(list(grads.values()), limit)
        for name in matrices:
            momentum[name].mul_(0.9).add_(grads[name])
        for name, update in zip(matrices, T.orthogonalize([momentum[name] for name in matrices])):
            w[name].sub_(update, alpha=rate)
        for name in grads:
            if name not in momentum:
                w[name].sub_(grads[name], alpha=rate * 50)
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
