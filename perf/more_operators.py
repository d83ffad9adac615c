"""What a training step does around its products, over the sizes, layouts and element types it is done with: the token embedding with its gradient,
the step from one block to the next (norm of the block's result, gate, residual sum, norm for the block that follows) with its gradients, and the
orthogonalised update of weight matrices by Newton-Schulz products.

A case is a dict with a "kind" (one of the keys of KINDS) and that kind's sizes and options. `listed` names twelve of them, `draw` makes another one
of the same ranges, `prepare` puts the operands on the device, `run` is one pass (the framework's operators where `own` is true, their plain form in
elementary torch operations where it is not), `work` counts what the pass cannot do without, and `exact` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF16, "f32": F32}
NO_TOKEN = -1       # the id of a position that has no token
EPS = 1e-6          # of the norms
STEPS, COEFFICIENTS, TINY = 5, (3.4445, -4.7750, 2.0315), 1e-7      # of the orthogonalisation

own = False


def listed():
    return [
        # a large model's embedding in training: 8192 tokens at once, the gradient of the whole table
        dict(name="embed_8192x131072", kind="embed", dtype="bf16", n=8192, d=4096, v=131072, ids="i64", padded=0.0, scale=1.0, grad=True),
        # a padded batch over a vocabulary of no round size, scaled by the root of the features as such models do
        dict(name="embed_padded_50021", kind="embed", dtype="bf16", n=3001, d=2048, v=50021, ids="i64", padded=0.3, scale=45.25, grad=True),
        # a small f32 model's table, rows of no whole 16 bytes
        dict(name="embed_f32_odd", kind="embed", dtype="f32", n=515, d=777, v=10007, ids="i32", padded=0.0, scale=1.0, grad=True),
        # decoding: one token for each of 64 sequences, latency
        dict(name="embed_64_tokens", kind="embed", dtype="bf16", n=64, d=4096, v=131072, ids="i64", padded=0.0, scale=1.0, grad=False),
        # between two blocks of a large model in training, both norms and a learned gate per channel: bound by the bytes
        dict(name="norms_8192x4096", kind="norms", stream="bf16", block="bf16", b=4, s=2048, d=4096, post=True, gate="channel", scale=1.0, grad=True),
        # an f32 residual stream beside bf16 blocks, a gate per sample, a scaled residual, rows of no whole 16 bytes
        dict(name="norms_sample_gate", kind="norms", stream="f32", block="bf16", b=7, s=331, d=1025, post=False, gate="sample", scale=0.5, grad=True),
        # a small f32 model, no gate: launches and latency
        dict(name="norms_small_f32", kind="norms", stream="f32", block="f32", b=2, s=48, d=256, post=True, gate="none", scale=1.0, grad=True),
        # decoding: one row, forward only
        dict(name="norms_1_row", kind="norms", stream="bf16", block="bf16", b=1, s=1, d=4096, post=True, gate="channel", scale=1.0, grad=False),
        # the update of a large gated block's weight matrix
        dict(name="orth_4096x14336", kind="orth", dtype="f32", b=1, m=4096, n=14336),
        # the three weight matrices of a middling block, one stack
        dict(name="orth_3x1024x2816", kind="orth", dtype="bf16", b=3, m=1024, n=2816),
        # a small f32 model's matrix, taller than wide, of odd extents
        dict(name="orth_703x255", kind="orth", dtype="f32", b=1, m=703, n=255),
        # one matrix for each of 64 heads
        dict(name="orth_64x128x128", kind="orth", dtype="bf16", b=64, m=128, n=128),
    ]


# ---------------------------------------------------------------------------------------------------------------- embedding
def _draw_embed(rng):
    dtype = rng.choice(["bf16", "bf16", "f32"])
    d = _up(_log(rng, 32, 4096), rng.choice([64, 8, 1]))
    return dict(kind="embed", dtype=dtype, n=_log(rng, 1, 16384), d=d, v=_log(rng, 100, 131072), ids=rng.choice(["i32", "i64"]),
                padded=rng.choice([0.0, 0.0, 0.3]), scale=rng.choice([1.0, 1.0, math.sqrt(d)]), grad=rng.random() < 0.75)


def _prepare_embed(c, g):
    n, d, v, dt = c["n"], c["d"], c["v"], TYPES[c["dtype"]]
    # the first ids are the frequent ones, falling as 1 / (id + 1)
    ids = (torch.rand((n,), generator=g, device="cuda", dtype=torch.float64) * math.log(v + 1)).exp_().sub_(1.0).long().clamp_(0, v - 1)
    if c["padded"]:
        ids = torch.where(torch.rand((n,), generator=g, device="cuda") < c["padded"], torch.full_like(ids, NO_TOKEN), ids)
    state = dict(table=_normal(g, (v, d), dt, 0.02), ids=ids.to(torch.int32) if c["ids"] == "i32" else ids)
    if c["grad"]:
        state["dy"] = _normal(g, (n, d), dt, 1e-3)
    return state


def _own_embed(c, s):
    from mimir_b200 import tensor as T
    ignore = NO_TOKEN if c["padded"] else None
    out = T.embedding(s["table"], s["ids"], scale=c["scale"], ignore_index=ignore)
    if not c["grad"]:
        return out
    return out, T.embedding_grad(s["dy"], s["ids"], c["v"], scale=c["scale"], ignore_index=ignore)


def _plain_embed(c, s):
    table, ids = s["table"], s["ids"].long()
    there = ids != NO_TOKEN
    at = torch.where(there, ids, torch.zeros_like(ids))
    factor = (there.to(F32) * c["scale"]).unsqueeze(1)
    out = (table[at].to(F32) * factor).to(table.dtype)
    if not c["grad"]:
        return out
    total = torch.zeros(table.shape, dtype=F32, device=table.device)
    total.index_add_(0, at, s["dy"].to(F32) * factor)
    return out, total.to(table.dtype)


def _exact_embed(c, s):
    ids = s["ids"].long()
    there = (ids >= 0).nonzero().squeeze(1)
    out = torch.zeros((c["n"], c["d"]), dtype=torch.float64, device="cuda")
    out[there] = s["table"].double()[ids[there]] * c["scale"]
    if not c["grad"]:
        return out
    # tokens in order of their classes: a class's sum is a difference of places in the sorted list
    order = there[torch.argsort(ids[there], stable=True)]
    classes, counts = torch.unique_consecutive(ids[order], return_counts=True)
    grad = torch.zeros((c["v"], c["d"]), dtype=torch.float64, device="cuda")
    if len(classes):
        grad[classes] = torch.segment_reduce(s["dy"].double()[order], "sum", lengths=counts, axis=0) * c["scale"]
    return out, grad


def _work_embed(c):
    size, tokens = _size(c["dtype"]), c["n"] * (1.0 - c["padded"])
    ids = c["n"] * (4 if c["ids"] == "i32" else 8)
    k = np.arange(c["v"], dtype=np.float64)
    share = np.log1p(1.0 / (k + 1.0)) / math.log(c["v"] + 1)
    rows = float((-np.expm1(tokens * np.log1p(-share))).sum())      # classes that are met at all
    nbytes, flops = size * c["d"] * (rows + c["n"]) + ids, c["n"] * c["d"]
    if c["grad"]:
        nbytes, flops = nbytes + size * c["d"] * (tokens + c["v"]) + ids, flops + 2 * tokens * c["d"]
    return nbytes, flops


# ------------------------------------------------------------------------------------------------- from one block to the next
def _draw_norms(rng):
    stream, block = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
    return dict(kind="norms", stream=stream, block=block, b=_log(rng, 1, 8), s=_log(rng, 1, 2048), d=_up(_log(rng, 32, 8192), rng.choice([64, 8, 1])),
                post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "sample"]), scale=rng.choice([1.0, 1.0, 0.5]), grad=rng.random() < 0.75)


def _prepare_norms(c, g):
    b, s, d, stream, block = c["b"], c["s"], c["d"], TYPES[c["stream"]], TYPES[c["block"]]
    about_one = lambda shape, dt: _normal(g, shape, F32, 0.2).add_(1.0).to(dt)  # noqa: E731
    state = dict(r=_normal(g, (b, s, d), stream, 3.0), h=_normal(g, (b, s, d), block, 0.7), gamma=about_one((d,), stream))
    state["post_gamma"] = about_one((d,), stream) if c["post"] else None
    state["gate"] = None if c["gate"] == "none" else _normal(g, (d,) if c["gate"] == "channel" else (b, 1, d), block, 0.5)
    if c["grad"]:
        state.update(dr=_normal(g, (b, s, d), stream, 1e-3), dx=_normal(g, (b, s, d), block, 3e-3))
    return state


def _own_norms(c, s):
    from mimir_b200 import tensor as T
    more = dict(post_gamma=s["post_gamma"], gate=s["gate"])
    if not c["grad"]:
        return T.residual_rmsnorm(s["r"], s["h"], s["gamma"], EPS, residual_scale=c["scale"], **more)
    r, x, kept = T.residual_rmsnorm_fwd(s["r"], s["h"], s["gamma"], EPS, residual_scale=c["scale"], **more)
    grads = T.residual_rmsnorm_bwd(s["dr"], s["dx"], s["r"], s["h"], s["gamma"], kept, **more)
    return (r, x) + tuple(t for t in grads if t is not None)


def _plain_norms(c, s):
    stream, block, d = s["r"].dtype, s["h"].dtype, c["d"]
    r, h, gamma = s["r"].to(F32), s["h"].to(F32), s["gamma"].to(F32)
    hat, factor = h, torch.ones((), dtype=F32, device=h.device)
    if c["post"]:
        inverse_h = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS)
        hat, factor = h * inverse_h, s["post_gamma"].to(F32)
    gate = torch.ones((), dtype=F32, device=h.device) if s["gate"] is None else s["gate"].to(F32)
    u = hat * factor
    new = c["scale"] * r + gate * u
    inverse = 1.0 / torch.sqrt((new * new).sum(-1, keepdim=True) / d + EPS)
    normed = new * inverse
    out = new.to(stream), (normed * gamma).to(block)
    if not c["grad"]:
        return out
    dx = s["dx"].to(F32)
    t = dx * gamma
    dnew = s["dr"].to(F32) + inverse * (t - normed * ((t * normed).sum(-1, keepdim=True) / d))
    dgamma = (dx * normed).sum((0, 1))
    du = dnew * gate
    dhat = du * factor
    dh = inverse_h * (dhat - hat * ((dhat * hat).sum(-1, keepdim=True) / d)) if c["post"] else dhat
    out += ((c["scale"] * dnew).to(stream), dh.to(block), dgamma.to(stream))
    if c["post"]:
        out += ((du * hat).sum((0, 1)).to(stream),)
    if s["gate"] is not None:
        each = dnew * u
        out += ((each.sum((0, 1)) if c["gate"] == "channel" else each.sum(1, keepdim=True)).to(block),)
    return out


def _exact_norms(c, s):
    names = ["r", "h", "gamma"] + ["post_gamma"] * c["post"] + ["gate"] * (c["gate"] != "none")
    with torch.enable_grad():
        p = {k: s[k].double().requires_grad_() for k in names}
        norm = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w  # noqa: E731
        u = norm(p["h"], p["post_gamma"]) if c["post"] else p["h"]
        new = p["r"] * c["scale"] + (u if c["gate"] == "none" else u * p["gate"])
        x = norm(new, p["gamma"])
        out = new.detach(), x.detach()
        if c["grad"]:
            out += torch.autograd.grad((new, x), [p[k] for k in names], (s["dr"].double(), s["dx"].double()))
    return out


def _work_norms(c):
    cells, a, b = c["b"] * c["s"] * c["d"], _size(c["stream"]), _size(c["block"])
    rows = 1 + c["post"]
    weights = a * c["d"] * rows + b * c["d"] * {"none": 0, "channel": 1, "sample": c["b"]}[c["gate"]]
    if not c["grad"]:
        return cells * 2 * (a + b) + weights, 10 * cells
    # forward: r and h to r and x; backward: dr, dx, r and h to dr and dh
    return cells * 5 * (a + b) + 3 * weights, 35 * cells


# ------------------------------------------------------------------------------------------------------ orthogonalised update
def _draw_orth(rng):
    m, n = _log(rng, 16, 4096), _log(rng, 16, 14336)
    if rng.random() < 0.5:
        m, n = _up(m, 64), _up(n, 64)
    if rng.random() < 0.4:
        m, n = n, m
    return dict(kind="orth", dtype=rng.choice(["bf16", "f32"]), b=_log(rng, 1, max(1, min(64, 2 ** 26 // (m * n)))), m=m, n=n)


def _prepare_orth(c, g):
    b, m, n, dt = c["b"], c["m"], c["n"], TYPES[c["dtype"]]
    # a gradient's momentum: directions that fall off, and noise below them
    k = min(m, n, 64)
    fall = torch.arange(1, k + 1, device="cuda", dtype=F32) ** -0.5
    x = torch.baddbmm(_normal(g, (b, m, n), F32, 0.3), _normal(g, (b, m, k), F32, 1.0) * fall, _normal(g, (b, k, n), F32, 1.0), beta=1.0, alpha=1.0)
    return dict(x=(x * 1e-3).to(dt))


def _own_orth(c, s):
    from mimir_b200 import tensor as T
    return T.orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=TINY)


def _plain_orth(c, s):
    x = s["x"].to(F32)
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + TINY)
    p, q, r = COEFFICIENTS
    for _ in range(STEPS):
        if c["m"] <= c["n"]:
            a = torch.matmul(x, x.mT)
            x = p * x + torch.matmul(q * a + r * torch.matmul(a, a), x)
        else:
            a = torch.matmul(x.mT, x)
            x = p * x + torch.matmul(x, q * a + r * torch.matmul(a, a))
    return x.to(BF16)


def _exact_orth(c, s):
    x = s["x"].double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + TINY)
    x = x if c["m"] <= c["n"] else x.mT
    p, q, r = COEFFICIENTS
    for _ in range(STEPS):
        # the even polynomial by Horner's rule on x x^T
        a = x @ x.mT
        f = a @ (r * a)
        f.diagonal(dim1=-2, dim2=-1).add_(p)
        x = f.add_(a, alpha=q) @ x
    return x if c["m"] <= c["n"] else x.mT


def _work_orth(c):
    k, l = sorted((c["m"], c["n"]))
    # x x^T and its square are symmetric: half of each; then the product with x
    return c["b"] * c["m"] * c["n"] * (_size(c["dtype"]) + 2), c["b"] * STEPS * (k * k * l + k * k * k + 2 * k * k * l)


# ------------------------------------------------------------------------------------------------------------------- common
KINDS = {
    "embed": (_draw_embed, _prepare_embed, _own_embed, _plain_embed, _work_embed, _exact_embed),
    "norms": (_draw_norms, _prepare_norms, _own_norms, _plain_norms, _work_norms, _exact_norms),
    "orth": (_draw_orth, _prepare_orth, _own_orth, _plain_orth, _work_orth, _exact_orth),
}


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _up(v, to):
    return (v + to - 1) // to * to


def _size(name):
    return 2 if name == "bf16" else 4


def _normal(g, shape, dtype, std):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def draw(rng):
    largest = {c["kind"]: c for c in reversed(listed())}        # (each kind's first)
    while True:
        c = KINDS[rng.choice(["embed", "norms", "orth"])][0](rng)
        w, most = work(c), work(largest[c["kind"]])
        if w["bytes"] <= 1.5 * most["bytes"] and (c["kind"] != "orth" or w["flops"] <= most["flops"]):
            return c


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = KINDS[case["kind"]][1](case, g)
    state["case"] = case
    return state


def run(state):
    c = state["case"]
    return KINDS[c["kind"]][2 if own else 3](c, state)


def work(case):
    nbytes, flops = KINDS[case["kind"]][4](case)
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    """What `run` returns for these inputs, from the operators' definitions in 64 bits."""
    return KINDS[case["kind"]][5](case, prepare(case, seed))
