"""A training step's own operators, over the sizes, layouts, masks and element types they are used with: the gated MLP block with its
gradients, the softmax cross-entropy of a linear output layer with its gradients, and the global norm of a list of gradients with
their clipping.

A case is a dict with a "kind" (one of the keys of KINDS) and that kind's sizes and options. `listed` names eleven of them, `draw` makes
another one of the same ranges, `prepare` puts the operands on the device, `run` is one pass (the framework's operators where `own`
is true, their plain form in elementary torch operations where it is not), `work` counts what the pass cannot do without, and `exact`
is the definition in 64 bits.
"""
import math

import torch
import torch.nn.functional as F

BF16, F32 = torch.bfloat16, torch.float32
IGNORED = -100      # the target of a position that has none

own = False


def listed():
    return [
        # forward and backward of a large model's gated MLP block: 8192 tokens at once
        dict(name="mlp_8192", kind="mlp", m=8192, k=4096, f=14336, n=4096, nk=False),
        # the same weights with a micro-batch of 64 tokens: bound by the weights' and the gradients' bytes
        dict(name="mlp_64_tokens", kind="mlp", m=64, k=4096, f=14336, n=4096, nk=False),
        # a middling block over a packed batch of an odd number of tokens, weights stored [out, in]
        dict(name="mlp_1777_tokens", kind="mlp", m=1777, k=1024, f=2816, n=1024, nk=True),
        # a small model's block: launches and latency
        dict(name="mlp_small", kind="mlp", m=96, k=256, f=704, n=256, nk=True),
        # the output layer of a large model in training: loss and gradients of 8192 tokens over 131072 classes
        dict(name="ce_8192x131072", kind="ce", dtype="bf16", n=8192, d=4096, v=131072, vd=True, masked=0.0, grad=True),
        # fine-tuning: half of the positions have no target (the prompts), a vocabulary of no round size
        dict(name="ce_masked_50021", kind="ce", dtype="bf16", n=3001, d=2048, v=50021, vd=True, masked=0.5, grad=True),
        # scoring one token at a time: the loss alone, bound by the weights' bytes
        dict(name="ce_score_1_token", kind="ce", dtype="bf16", n=1, d=4096, v=131072, vd=True, masked=0.0, grad=False),
        # a small f32 model's output layer, weights stored [in, out]
        dict(name="ce_f32_10007", kind="ce", dtype="f32", n=512, d=784, v=10007, vd=False, masked=0.0, grad=True),
        # gradients of the f32 MLP 784 / 1024 / 1024 / 10, weights and biases: six tensors, launches and latency
        dict(name="clip_small_f32", kind="clip", dtype="f32", count=6, largest=1024 * 1024, smallest=10, over=True, packed=False),
        # bf16 gradients of several transformer blocks, one per weight
        dict(name="clip_blocks_bf16", kind="clip", dtype="bf16", count=24, largest=14336 * 4096, smallest=4096, over=True, packed=False),
        # many tensors packed end to end in one buffer at whatever offset they come to, with a norm below the limit
        dict(name="clip_packed_f32", kind="clip", dtype="f32", count=700, largest=3000000, smallest=1, over=False, packed=True),
    ]


# ------------------------------------------------------------------------------------------------------------ gated MLP block
def _draw_mlp(rng):
    to = rng.choice([64, 8, 1])     # whole tiles, rows of whole 16 bytes, or neither
    k, f, n = (_up(_log(rng, lo, hi), to) for lo, hi in ((64, 4096), (128, 14336), (64, 4096)))
    return dict(kind="mlp", m=_log(rng, 1, 8192), k=k, f=f, n=n, nk=rng.random() < 0.5)


def _prepare_mlp(c, g):
    def weight(i, o):
        return _normal(g, (o, i), BF16, 0.02).t() if c["nk"] else _normal(g, (i, o), BF16, 0.02)
    return dict(x=_normal(g, (c["m"], c["k"]), BF16, 1.0), w1=weight(c["k"], c["f"]), w3=weight(c["k"], c["f"]), w2=weight(c["f"], c["n"]),
                dy=_normal(g, (c["m"], c["n"]), BF16, 1e-3))


def _own_mlp(c, s):
    from mimir_b200 import tensor as T
    y, kept = T.mlp_gated_fwd(s["x"], s["w1"], s["w3"], s["w2"])
    return (y,) + tuple(T.mlp_gated_bwd(s["dy"], s["x"], s["w1"], s["w3"], s["w2"], kept))


def _plain_mlp(c, s):
    x, w1, w3, w2, dy = (s[k].to(F32) for k in ("x", "w1", "w3", "w2", "dy"))
    a, b = x @ w1, x @ w3
    e = 1.0 / (1.0 + torch.exp(-a))
    gate = a * e
    h = gate * b
    dh = dy @ w2.t()
    da, db = dh * b * (e + gate * (1.0 - e)), dh * gate
    return tuple(t.to(BF16) for t in (h @ w2, da @ w1.t() + db @ w3.t(), x.t() @ da, x.t() @ db, h.t() @ dy))


def _exact_mlp(c, s):
    x, w1, w3, w2 = (s[k].double().requires_grad_() for k in ("x", "w1", "w3", "w2"))
    with torch.enable_grad():
        y = (F.silu(x @ w1) * (x @ w3)) @ w2
        grads = torch.autograd.grad(y, (x, w1, w3, w2), s["dy"].double())
    return (y.detach(),) + grads


def _work_mlp(c):
    m, k, f, n = c["m"], c["k"], c["f"], c["n"]
    return 2 * (2 * m * k + 2 * m * n + 2 * (2 * k * f + f * n)), 6 * m * f * (2 * k + n)


# -------------------------------------------------------------------------------------- cross-entropy of a linear output layer
def _draw_ce(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    to = rng.choice([64, 8, 1])
    n, d, v = (_log(rng, 1, 8192), _log(rng, 64, 4096), _log(rng, 1000, 131072)) if dtype == "bf16" else (
        _log(rng, 1, 2048), _log(rng, 64, 1024), _log(rng, 100, 32768))
    return dict(kind="ce", dtype=dtype, n=n, d=_up(d, to), v=v, vd=rng.random() < 0.7, masked=rng.choice([0.0, 0.0, 0.3, 0.8]), grad=rng.random() < 0.7)


def _prepare_ce(c, g):
    dt, n, d, v = _dtype(c), c["n"], c["d"], c["v"]
    w = _normal(g, (v, d) if c["vd"] else (d, v), dt, 2.0 / math.sqrt(d))
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    if c["masked"]:
        t = torch.where(torch.rand((n,), generator=g, device="cuda") < c["masked"], torch.full_like(t, IGNORED), t)
    return dict(x=_normal(g, (n, d), dt, 1.0), w=w.t() if c["vd"] else w, t=t)


def _own_ce(c, s):
    from mimir_b200 import tensor as T
    ignore = IGNORED if c["masked"] else None
    if not c["grad"]:
        return T.linear_cross_entropy(s["x"], s["w"], s["t"], ignore_index=ignore, reduction="none", return_lse=True)
    return T.linear_cross_entropy_with_grad(s["x"], s["w"], s["t"], ignore_index=ignore, reduction="mean")


def _plain_ce(c, s):
    x, w, t = s["x"].to(F32), s["w"].to(F32), s["t"]
    logits = x @ w
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    kept = t != IGNORED
    at = torch.where(kept, t, torch.zeros_like(t)).unsqueeze(1)
    losses = torch.where(kept, lse - logits.gather(1, at).squeeze(1), torch.zeros_like(lse))
    lse = torch.where(kept, lse, torch.zeros_like(lse))
    if not c["grad"]:
        return losses, lse
    each = kept.to(F32) / kept.sum().clamp(min=1)
    p = e / total
    p.scatter_add_(1, at, torch.full_like(total, -1.0))
    p = p * each.unsqueeze(1)
    return (losses * each).sum(), (p @ w.t()).to(s["x"].dtype), (x.t() @ p).to(s["x"].dtype)


def _exact_ce(c, s):
    x, w, t = s["x"].double(), s["w"].double(), s["t"]
    kept = t != IGNORED
    count = max(int(kept.sum()), 1)
    losses, lses, dx, dw = [], [], [], torch.zeros_like(w)
    for i in range(0, c["n"], 2048):
        xi, ti, ki = x[i:i + 2048], t[i:i + 2048], kept[i:i + 2048]
        logits = xi @ w
        lse = torch.logsumexp(logits, 1)
        losses.append(F.cross_entropy(logits, ti, reduction="none", ignore_index=IGNORED))
        lses.append(lse.masked_fill(~ki, 0.0))
        if c["grad"]:
            p = torch.softmax(logits, 1)
            p[torch.arange(len(ti), device=ti.device)[ki], ti[ki]] -= 1.0
            p[~ki] = 0.0
            dx.append(p @ w.t() / count)
            dw.addmm_(xi.t(), p, alpha=1.0 / count)
    if not c["grad"]:
        return torch.cat(losses), torch.cat(lses)
    return torch.cat(losses).sum() / count, torch.cat(dx), dw


def _work_ce(c):
    n, d, v, size = c["n"], c["d"], c["v"], _size(c)
    kept = n * (1.0 - c["masked"])      # a position without a target needs no logits
    io = size * (kept * d + d * v) + 8 * n
    if not c["grad"]:
        return io + 8 * n, 2 * kept * d * v
    return io + size * (n * d + d * v) + 4, 6 * kept * d * v


# ------------------------------------------------------------------------------------------- norm and clipping of gradients
def _sizes(c):
    """The tensors' lengths: spread over their logarithm, no two neighbours alike, the largest and the smallest among them."""
    n = c["count"]
    stride = 7 if n % 7 else 11 if n % 11 else 13
    ratio = c["largest"] / c["smallest"]
    return [max(1, round(c["smallest"] * ratio ** ((stride * i) % n / max(n - 1, 1)))) for i in range(n)]


def _draw_clip(rng):
    while True:
        c = dict(kind="clip", dtype=rng.choice(["f32", "bf16"]), count=_log(rng, 1, 700), largest=_log(rng, 1000, 14336 * 4096),
                 smallest=_log(rng, 1, 1000), over=rng.random() < 0.5, packed=False)
        c["packed"] = c["count"] > 30 or rng.random() < 0.3
        if sum(_sizes(c)) * _size(c) <= 6e8:
            return c


def _prepare_clip(c, g):
    sizes, dt = _sizes(c), _dtype(c)
    total = sum(sizes)
    std = 1e-2
    limit = std * math.sqrt(total) * (0.1 if c["over"] else 3.0)
    if not c["packed"]:
        grads = [_normal(g, (s,), dt, std) for s in sizes]
        return dict(grads=grads, limit=limit, out=[torch.empty_like(t) for t in grads])
    flat, out = _normal(g, (total,), dt, std), torch.empty((total,), dtype=dt, device="cuda")
    return dict(grads=list(flat.split(sizes)), limit=limit, out=list(out.split(sizes)), whole=out)


def _own_clip(c, s):
    from mimir_b200 import tensor as T
    norm = T.clip_grad_norm(s["grads"], s["limit"], out=s["out"])
    return norm, s["whole"] if c["packed"] else s["out"]


def _plain_clip(c, s):
    flat = torch.cat([t.to(F32) for t in s["grads"]])
    norm = torch.sqrt((flat * flat).sum())
    flat = (flat * torch.clamp(s["limit"] / (norm + 1e-6), max=1.0)).to(_dtype(c))
    return norm, flat if c["packed"] else list(flat.split([t.numel() for t in s["grads"]]))


def _exact_clip(c, s):
    flat = torch.cat([t.double() for t in s["grads"]])
    norm = torch.linalg.vector_norm(flat)
    flat = flat * min(1.0, s["limit"] / (float(norm) + 1e-6))
    return norm, flat if c["packed"] else list(flat.split([t.numel() for t in s["grads"]]))


def _work_clip(c):
    total = sum(_sizes(c))
    return 2 * _size(c) * total + 4, 3 * total


# ------------------------------------------------------------------------------------------------------------------- common
KINDS = {
    "mlp": (_draw_mlp, _prepare_mlp, _own_mlp, _plain_mlp, _work_mlp, _exact_mlp),
    "ce": (_draw_ce, _prepare_ce, _own_ce, _plain_ce, _work_ce, _exact_ce),
    "clip": (_draw_clip, _prepare_clip, _own_clip, _plain_clip, _work_clip, _exact_clip),
}


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _up(v, to):
    return (v + to - 1) // to * to


def _dtype(c):
    return BF16 if c.get("dtype", "bf16") == "bf16" else F32


def _size(c):
    return 2 if _dtype(c) == BF16 else 4


def _normal(g, shape, dtype, std):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def draw(rng):
    while True:
        c = KINDS[rng.choice(["mlp", "mlp", "ce", "ce", "clip"])][0](rng)
        w = work(c)
        # none costs more than the largest listed one; f32 products take several times as long for the same count
        if w["flops"] <= (1e12 if c.get("dtype") == "f32" else 2.6e13):
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
