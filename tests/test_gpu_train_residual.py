"""The step from one block to the next (norms, gate, residual sum) and its gradients against the formulas in 64 bits, through the public operators.

Tolerances. u = 2^-8 (bf16) or 2^-24 (f32) is half a step of a result's type, and every result is rounded to it once. Before that, in f32 (half a step e = 2^-24):
a sum of a row's d squares is off by less than 42 e of itself (up to 32 values by a thread, two joins of 5 steps), the inverse root by half of that and by the roundings of the mean, eps, root and
quotient: under 32 e = C of itself. A sum of products of a row is off by 42 e of the sum of the magnitudes, beside what its terms are off. The bounds below follow each formula's
terms with their magnitudes: a product adds its factors' relative errors and e, a sum its terms' errors and e of its magnitude. A sum of n rows adds n e of the sum of the magnitudes."""
import itertools

import pytest
import torch

from util import randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
E = 2.0 ** -24
C = 32 * E
EPS = 1e-6


def inputs(shape, stream, block, post, gate, seed=0, weights=None):
    lead, d = shape[:-1], shape[-1]
    w = weights or stream
    about = lambda s, k, dt: (randn(s, k, 0.2) + 1).to(dt)  # noqa: E731
    p = dict(r=randn(shape, seed, 2.0, stream), h=randn(shape, seed + 1, 0.7, block), gamma=about((d,), seed + 2, w))
    p["post_gamma"] = about((d,), seed + 3, w) if post else None
    p["gate"] = None if gate is None else randn((d,) if gate == 0 else (*lead[:gate], *(1,) * (len(lead) - gate), d), seed + 4, 0.5, block)
    return p, randn(shape, seed + 5, 1.0, stream), randn(shape, seed + 6, 1.0, block)


def formulas(p, dr, dx, a, b, eps=EPS):
    """{name: (value, bound before the last rounding)} in 64 bits."""
    r, h, gamma = (None if p[k] is None else p[k].double() for k in ("r", "h", "gamma"))
    one = torch.ones((), dtype=torch.float64, device=r.device)
    gate = one if p["gate"] is None else p["gate"].double()
    f = one if p["post_gamma"] is None else p["post_gamma"].double()
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    out = {}
    if h is None:
        e, hat, new, err = one, one * 0, r, r.abs() * 0
        q = one * 0
    else:
        e = one if p["post_gamma"] is None else 1 / (mean(h * h) + eps).sqrt()
        hat, q = h * e, b * gate * f
        new = a * r + q * hat
        size = (a * r).abs() + (q * hat).abs()
        err = (C + 6 * E) * size
        out["r"] = new, err
    if gamma is None:
        gamma, s, cs = one * 0, one, one * 0
    else:
        s = 1 / (mean(new * new) + eps).sqrt()
        cs = C + (mean(err * err) / mean(new * new).clamp(min=1e-300)).sqrt()          # what s is off, of itself
        out["x"] = new * s * gamma, (s * gamma).abs() * err + (new * s * gamma).abs() * (cs + 3 * E)
    if dr is None and dx is None:
        return out
    dr = one * 0 if dr is None else dr.double()
    dx = one * 0 if dx is None else dx.double()
    rhat = new * s
    erhat = s * err + rhat.abs() * (cs + 3 * E)
    t = dx * gamma
    m = mean(t * rhat)
    em = mean(t.abs() * erhat) + (42 + 4) * E * mean((t * rhat).abs())
    D = dr + s * (t - rhat * m)
    # D and, the same way, what the second mean is of: k = s m
    eD = 4 * E * dr.abs() + (s * t).abs() * (cs + 6 * E) + s * (erhat * m.abs() + rhat.abs() * em + (rhat * m).abs() * (cs + 6 * E))
    sizeD = dr.abs() + (s * t).abs() + s * (rhat * m).abs()
    eD = eD + 4 * E * sizeD
    out["dr"] = a * D, abs(a) * (eD + 2 * E * D.abs())
    ehat = hat.abs() * (C + 2 * E)
    if p["h"] is not None:
        if p["post_gamma"] is None:
            dh, edh = q * D, q.abs() * (eD + 4 * E * D.abs())
        else:
            n2 = mean(q * hat * D)
            en2 = mean(q.abs() * (ehat * sizeD + hat.abs() * eD)) + (42 * 2 + 12) * E * mean(q.abs() * hat.abs() * sizeD)
            dh = e * (q * D - hat * n2)
            edh = e * (q.abs() * eD + ehat * n2.abs() + hat.abs() * en2) + (C + 8 * E) * e * ((q * D).abs() + (hat * n2).abs())
        out["dh"] = dh, edh
    rows = tuple(range(r.dim() - 1))
    n = max(1, r.numel() // max(1, r.shape[-1]))

    def over_rows(v, err, like):
        axes = tuple(i for i in range(v.dim() - 1) if i >= v.dim() - like.dim() and like.shape[i - v.dim()] == 1 or i < v.dim() - like.dim())
        return (v.sum(axes, keepdim=True).reshape(like.shape) if axes else v, ((err + (n + 4) * E * v.abs()).sum(axes, keepdim=True).reshape(like.shape) if axes else err + 4 * E * v.abs()))

    if p["gamma"] is not None:
        out["dgamma"] = over_rows(dx * rhat, dx.abs() * erhat, p["gamma"])
    if p["post_gamma"] is not None:
        w = b * gate
        out["dpost_gamma"] = over_rows(w * D * hat, w.abs() * (eD * hat.abs() + D.abs() * ehat), p["post_gamma"])
    if p["gate"] is not None:
        w = b * f
        out["dgate"] = over_rows(w * D * hat, w.abs() * (eD * hat.abs() + D.abs() * ehat), p["gate"])
    return out


def same_bits(a, b):
    return torch.equal(*(t.view(torch.int16 if t.dtype == BF16 else torch.int32) for t in (a, b)))


def run(p, dr, dx, a, b, eps=EPS):
    from mimir_b200 import tensor as T
    more = dict(post_gamma=p["post_gamma"], gate=p["gate"])
    new, x, kept = T.residual_rmsnorm_fwd(p["r"], p["h"], p["gamma"], eps, residual_scale=a, branch_scale=b, **more)
    plain = T.residual_rmsnorm(p["r"], p["h"], p["gamma"], eps, residual_scale=a, branch_scale=b, **more)
    assert same_bits(plain[0], new) and (x is None) == (plain[1] is None) and (x is None or same_bits(plain[1], x))
    grads = T.residual_rmsnorm_bwd(dr, dx if p["gamma"] is not None else None, p["r"], p["h"], p["gamma"], kept, **more)
    T.device_status()
    got = dict(r=new if p["h"] is not None else None, x=x, **dict(zip(("dr", "dh", "dgamma", "dpost_gamma", "dgate"), grads)))
    return {k: v for k, v in got.items() if v is not None}


def check(p, dr, dx, a=1.0, b=1.0):
    got, want = run(p, dr, dx, a, b), formulas(p, dr, dx if p["gamma"] is not None else None, a, b)
    assert got.keys() == want.keys()
    like = dict(r=p["r"], x=p["r"] if p["h"] is None else p["h"], dr=p["r"], dh=p["h"], dgamma=p["gamma"], dpost_gamma=p["post_gamma"], dgate=p["gate"])
    for k, g in got.items():
        v, bound = want[k]
        assert g.shape == like[k].shape and g.dtype == like[k].dtype, k
        bound = 1.02 * (bound + U[g.dtype] * (v.abs() + bound)) + 1e-37
        assert bool(((g.double() - v).abs() <= bound).all()), (k, float(((g.double() - v).abs() / bound).max()))
    return got


TYPES = [(BF16, BF16), (F32, BF16), (F32, F32)]
# one value; around a warp's and a block's columns; rows of no whole 16 bytes; each number of columns a thread holds
SHAPES = [(1, 1), (1, 8), (3, 5), (2, 31), (9, 32), (5, 33), (7, 255), (130, 256), (6, 264), (65, 777), (3, 1025), (40, 2048), (9, 2049), (33, 2056), (301, 4096),
          (11, 8191), (4, 8192), (3, 8200), (2, 16385), (5, 32768), (2, 32767)]


@pytest.mark.parametrize("shape,types", list(itertools.product(SHAPES, TYPES)))
def test_both_norms_and_a_gate(shape, types):
    check(*inputs(shape, *types, True, 0), a=0.75, b=1.5)


@pytest.mark.parametrize("post,gate,types", list(itertools.product([False, True], [None, 0, 1, 2], TYPES)))
def test_every_combination(post, gate, types):
    for d in (520, 321):
        check(*inputs((3, 50, d), *types, post, gate), a=-0.5)


@pytest.mark.parametrize("lead,gate", [((1, 1), 1), ((7, 1), 1), ((1, 9), 1), ((200, 3), 1), ((2, 700), 1), ((2, 3, 40), 1), ((2, 3, 40), 2), ((500,), 1), ((3, 301), 2), ((1500, 2), 1)])
def test_gates_of_runs_of_rows(lead, gate):
    """More and fewer groups of rows than there are blocks, groups of one row, one group."""
    check(*inputs((*lead, 264), F32, BF16, True, gate))


@pytest.mark.parametrize("d,gate", list(itertools.product([4104, 5001, 8192, 8200, 8193, 17088, 30008], [None, 0, 1, 2])))
def test_long_rows(d, gate):
    """Rows that are read twice: sums for their columns in shared memory and outside, for all rows and for groups of them, more rows than blocks."""
    for lead, types, post in (((2, 5), (F32, F32), True), ((3, 101), (BF16, BF16), gate != 1)):
        check(*inputs((*lead, d), *types, post, gate), a=-0.5)


@pytest.mark.parametrize("d,gate", list(itertools.product([8, 100, 1024, 4099], [None, 0, 1, 2])))
def test_rows_that_begin_elsewhere(d, gate):
    """Tensors that do not start on 16 bytes, by every kind of gate."""
    p, dr, dx = inputs((3, 301, d), BF16, BF16, True, gate)

    def moved(t):
        return None if t is None else torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    check({k: moved(t) for k, t in p.items()}, moved(dr), moved(dx), b=0.5)


@pytest.mark.parametrize("weights", [F32, BF16])
def test_weights_of_either_type(weights):
    check(*inputs((70, 512), F32, BF16, True, 0, weights=weights))
    check(*inputs((70, 100), BF16, BF16, True, 0, weights=weights))


@pytest.mark.parametrize("types", TYPES)
def test_the_norm_alone(types):
    for shape in ((5, 8), (300, 4096), (2, 3, 777)):
        p, dr, dx = inputs(shape, types[0], types[0], False, None)
        p["h"] = None
        got = check(p, dr, dx)
        assert "dh" not in got
        check(p, None, dx)


def test_no_norm_after():
    for post in (False, True):
        p, dr, dx = inputs((4, 33, 520), F32, BF16, post, 1)
        p["gamma"] = None
        check(p, dr, None, a=0.5, b=2.0)
        p, dr, dx = inputs((33, 520), F32, BF16, post, 0)
        check(p, None, dx)


def test_many_rows():
    check(*inputs((20000, 64), BF16, BF16, True, 0))
    check(*inputs((3000, 1032), F32, F32, True, 0))


@pytest.mark.parametrize("d,types", [(2048, (BF16, BF16)), (2049, (BF16, BF16)), (8200, (F32, BF16))])
def test_rows_that_begin_past_32_bits(d, types):
    """More than 2^31 values, of which the last rows are compared with a call of their own: whole rows, ragged ones, and those held in registers. Bits, where both calls have a row's
    columns in the same places; else within what both may be off."""
    from mimir_b200 import tensor as T
    n, few = 2 ** 31 // d + 24, 16
    p, _, _ = inputs((few, d), *types, False, 0)
    p["post_gamma"] = p["gamma"]
    last = torch.zeros((n, d), dtype=types[0], device="cuda")
    r, h, dr, dx = last, *(torch.zeros((n, d), dtype=t, device="cuda") for t in (types[1], types[0], types[1]))
    for k, (t, of) in enumerate(((r, p["r"]), (h, p["h"]), (dr, None), (dx, None))):
        t[-few:] = of if of is not None else randn((few, d), 30 + k, 1.0, t.dtype)
    own = dict(p, r=r[-few:].clone(), h=h[-few:].clone())
    want = run(own, dr[-few:].clone(), dx[-few:].clone(), 1.0, 1.0)
    more = dict(post_gamma=p["post_gamma"], gate=p["gate"])
    new, x, kept = T.residual_rmsnorm_fwd(r, h, p["gamma"], EPS, **more)
    got = dict(r=new[-few:].clone(), x=x[-few:].clone())
    assert not bool(new[:64].any()) and not bool(x[:64].any())
    del new, x
    got.update(zip(("dr", "dh", "dgamma", "dpost_gamma", "dgate"), T.residual_rmsnorm_bwd(dr, dx, r, h, p["gamma"], kept, **more)))
    assert not bool(got["dr"][:64].any()) and not bool(got["dh"][:64].any())
    got["dr"], got["dh"] = got["dr"][-few:].clone(), got["dh"][-few:].clone()
    bounds = formulas(own, dr[-few:], dx[-few:], 1.0, 1.0)
    for name, value in got.items():
        exact, off = bounds[name]
        assert bool(((value.double() - exact).abs() <= 1.02 * (off + U[value.dtype] * (exact.abs() + off)) + 1e-37).all()), name
        if d % 8 == 0 and name in ("r", "x", "dr", "dh"):
            assert same_bits(value, want[name]), name


def test_empty_extents():
    for shape in ((0, 16), (3, 0, 16), (4, 0)):
        p, dr, dx = inputs(shape, F32, BF16, True, 0)
        got = run(p, dr, dx, 1.0, 1.0)
        assert all(not bool(t.any()) for t in got.values()) and tuple(got["dgate"].shape) == tuple(p["gate"].shape)


def test_rows_of_zeros_and_values_that_are_not_finite():
    p, dr, dx = inputs((40, 264), BF16, BF16, True, 0)
    clean = run(p, dr, dx, 1.0, 1.0)
    p["r"][3] = p["h"][3] = 0
    check(p, dr, dx)
    p["r"][3] = 0.5
    p["h"][7, 5], p["r"][9, 0] = float("nan"), float("inf")
    got = run(p, dr, dx, 1.0, 1.0)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 7, 9]] = False
    for k in ("r", "x", "dr", "dh"):
        assert torch.equal(got[k][keep], clean[k][keep])
    assert bool(got["r"][7].isnan().all()) and bool(got["x"][7].isnan().all()) and bool(got["x"][9, 0].isnan())


def test_large_and_small_rows():
    """Rows whose squares are as large and as small as f32 holds."""
    p, dr, dx = inputs((4, 512), F32, F32, True, 0)
    p["gate"] = None
    p["h"][0] *= 1e17
    p["h"][1] *= 1e-17       # (eps is more)
    p["r"][2] *= 1e17
    check(p, dr, dx)


def test_strides_and_addresses():
    p, dr, dx = inputs((6, 20, 256), F32, BF16, True, 1)
    want = run(p, dr, dx, 1.0, 1.0)

    def moved(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:].copy_(t.reshape(-1))
        return room[1:].view(t.shape)

    def wide(t):
        room = torch.full((*t.shape[:-1], t.shape[-1] + 8), float("nan"), dtype=t.dtype, device="cuda")
        room[..., :t.shape[-1]] = t
        return room[..., :t.shape[-1]]

    for k, t in run({k: wide(t) for k, t in p.items()}, wide(dr), wide(dx), 1.0, 1.0).items():
        assert torch.equal(t, want[k]), k
    check({k: moved(t) for k, t in p.items()}, moved(dr), moved(dx))
    # one operand off 16 bytes
    for name in p:
        check({**p, name: moved(p[name])}, dr, dx)


def test_same_bits_again_on_another_stream_and_in_a_graph():
    p, dr, dx = inputs((5, 301, 1032), BF16, BF16, True, 1)
    want = run(p, dr, dx, 1.0, 0.5)
    for _ in range(3):
        assert all(torch.equal(t, want[k]) for k, t in run(p, dr, dx, 1.0, 0.5).items())
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = run(p, dr, dx, 1.0, 0.5)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(t, want[k]) for k, t in got.items())
    from mimir_b200 import tensor as T
    more = dict(post_gamma=p["post_gamma"], gate=p["gate"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, x, kept = T.residual_rmsnorm_fwd(p["r"], p["h"], p["gamma"], EPS, branch_scale=0.5, **more)
        grads = T.residual_rmsnorm_bwd(dr, dx, p["r"], p["h"], p["gamma"], kept, **more)
    for t in (new, x, *grads):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip((new, x, *grads), want.values()))


def test_gradient_against_differences():
    """<r', dr> + <x, dx> along a step of each operand, f32: the quotient of two forward passes and the gradient's product, within the roundings of the two sums (their
    results' bounds) and the quotient's curvature, which the formulas give."""
    from mimir_b200 import tensor as T
    p, dr, dx = inputs((6, 40, 96), F32, F32, True, 1)
    a, b = 0.5, 1.5
    got = run(p, dr, dx, a, b)

    def loss(q):
        new, x = T.residual_rmsnorm(q["r"], q["h"], q["gamma"], EPS, post_gamma=q["post_gamma"], gate=q["gate"], residual_scale=a, branch_scale=b)
        return float((new.double() * dr.double()).sum() + (x.double() * dx.double()).sum())

    def exact(q):
        f = formulas(q, None, None, a, b)
        noise = sum(float(((f[k][1] + E * f[k][0].abs()) * w.double().abs()).sum()) for k, w in (("r", dr), ("x", dx)))
        return float((f["r"][0] * dr.double()).sum() + (f["x"][0] * dx.double()).sum()), noise

    want = formulas(p, dr, dx, a, b)
    for name, g in (("r", "dr"), ("h", "dh"), ("gamma", "dgamma"), ("post_gamma", "dpost_gamma"), ("gate", "dgate")):
        step = torch.sign(got[g]) * p[name].abs().mean() / 64
        plus, minus = {**p, name: p[name] + step}, {**p, name: p[name] - step}
        delta = plus[name].double() - minus[name].double()
        (up, noise_up), (down, noise_down) = exact(plus), exact(minus)
        slope = float((got[g].double() * delta).sum())
        curvature = abs(up - down - float((want[g][0] * delta).sum()))
        allowed = noise_up + noise_down + curvature + float(((want[g][1] + E * want[g][0].abs()) * delta.abs()).sum())
        assert abs(slope) > 4 * allowed, (name, "the step says nothing")
        assert abs(loss(plus) - loss(minus) - slope) <= allowed, name


def test_refusals():
    import ctypes as ct

    from mimir_b200 import MimkError, _lib
    from mimir_b200 import tensor as T
    p, dr, dx = inputs((6, 20, 64), F32, BF16, True, 1)
    r, h, gamma, post, gate = (p[k] for k in ("r", "h", "gamma", "post_gamma", "gate"))
    with pytest.raises(ValueError, match="one shape"):
        T.residual_rmsnorm(r, h[:5], gamma, EPS)
    with pytest.raises(TypeError):
        T.residual_rmsnorm(r.half(), h, gamma, EPS)
    with pytest.raises(TypeError, match="BF16 beside an F32"):
        T.residual_rmsnorm(r.to(BF16), h.float(), gamma, EPS)
    with pytest.raises(ValueError, match="gamma extent"):
        T.residual_rmsnorm(r, h, gamma[:63], EPS)
    with pytest.raises(ValueError, match="gamma extent"):
        T.residual_rmsnorm(r, h, gamma, EPS, post_gamma=gamma.repeat(20, 1))
    for bad in (gate[:, 0], gate[:5], gate[..., :63], torch.ones((20, 64), device="cuda"), torch.ones((1, 20, 64), device="cuda"), torch.ones((), device="cuda"),
                torch.ones((1, 6, 1, 64), device="cuda")):
        with pytest.raises(ValueError, match="the gate"):
            T.residual_rmsnorm(r, h, gamma, EPS, gate=bad)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            T.residual_rmsnorm(r, h, gamma, eps)
    for bad in (dict(post_gamma=post), dict(gate=gate), dict(residual_scale=0.5), dict(branch_scale=2.0)):
        with pytest.raises(ValueError, match="norm of r alone"):
            T.residual_rmsnorm(r, None, gamma, EPS, **bad)
    with pytest.raises(ValueError, match="norm of r alone"):
        T.residual_rmsnorm(r, None, None, EPS)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        T.residual_rmsnorm(r, h.cpu(), gamma, EPS)
    with pytest.raises(MimkError) as e:
        T.residual_rmsnorm(torch.ones((1, 32776), device="cuda"), None, torch.ones(32776, device="cuda"), EPS)
    assert e.value.status == 8
    _, _, kept = T.residual_rmsnorm_fwd(r, h, gamma, EPS, post_gamma=post, gate=gate)
    back = lambda *a, **k: T.residual_rmsnorm_bwd(*a, kept, **{**dict(post_gamma=post, gate=gate), **k})  # noqa: E731
    with pytest.raises(ValueError, match="other operands"):
        back(dr, dx, r, h, gamma, gate=None)
    with pytest.raises(ValueError, match="other operands"):
        back(dr[:2], dx[:2], r[:2], h[:2], gamma, gate=gate[:2])
    with pytest.raises(ValueError, match="dx is the gradient"):
        back(dr, None, r, h, gamma)
    with pytest.raises(ValueError, match="results' shape"):
        back(dr[:2], dx, r, h, gamma)
    with pytest.raises(TypeError):
        back(dr.to(BF16), dx, r, h, gamma)
    with pytest.raises(TypeError):
        back(dr, dx.float(), r, h, gamma)
    # the C entry points: addresses, and a workspace that is missing, too small or unaligned
    lib, need = _lib.lib(), ct.c_uint64()
    d, held, _, put = T._residual_desc("", r, h, gamma, post, gate, EPS, 1.0, 1.0)
    assert lib.mimk_residual_rmsnorm_fwd(ct.byref(d), None) == 1
    out = [torch.empty_like(t) for t in (r, h, gamma, post, gate)]
    put("dr_out", dr), put("dx", dx)
    d.kept = kept.buffer.data_ptr()
    d.dr, d.dh, d.dgamma, d.dpost_gamma, d.dgate = (t.data_ptr() for t in out)
    assert lib.mimk_residual_rmsnorm_workspace(ct.byref(d), ct.byref(need)) == 0 and need.value > 0
    assert lib.mimk_residual_rmsnorm_bwd(ct.byref(d), None) == 9
    room = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = room.data_ptr(), need.value - 1
    assert lib.mimk_residual_rmsnorm_bwd(ct.byref(d), None) == 9
    d.workspace, d.workspace_bytes = room.data_ptr() + 4, need.value
    assert lib.mimk_residual_rmsnorm_bwd(ct.byref(d), None) == 3
    d.workspace, d.dr = room.data_ptr(), out[0].data_ptr() + 2
    assert lib.mimk_residual_rmsnorm_bwd(ct.byref(d), None) == 3
    for name in ("dr", "dh", "dgamma", "dpost_gamma", "dgate", "kept"):
        d.dr, d.dh, d.dgamma, d.dpost_gamma, d.dgate, d.kept = (*(t.data_ptr() for t in out), kept.buffer.data_ptr())
        setattr(d, name, None)
        assert lib.mimk_residual_rmsnorm_bwd(ct.byref(d), None) == 1, name


def test_results_in_place():
    """r_out in r's place, and dr in dr_out's, through the C entry points."""
    import ctypes as ct

    from mimir_b200 import _lib
    from mimir_b200 import tensor as T
    p, dr, dx = inputs((30, 520), BF16, BF16, True, 0)
    want = run(p, dr, dx, 1.0, 1.0)
    d, held, _, put = T._residual_desc("", p["r"].clone(), p["h"], p["gamma"], p["post_gamma"], p["gate"], EPS, 1.0, 1.0)
    x, kept, room = torch.empty_like(p["h"]), torch.empty((2, 30), device="cuda"), torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    d.r_out, d.x, d.kept = d.r, x.data_ptr(), kept.data_ptr()
    assert _lib.lib().mimk_residual_rmsnorm_fwd(ct.byref(d), T._stream()) == 0
    assert torch.equal(held[0], want["r"]) and torch.equal(x, want["x"])
    held[0].copy_(p["r"])
    arrived = dr.clone()
    grads = [torch.empty_like(p[k]) for k in ("h", "gamma", "post_gamma", "gate")]
    d.dr_out = d.dr = arrived.data_ptr()
    d.dx = dx.data_ptr()
    d.dh, d.dgamma, d.dpost_gamma, d.dgate = (t.data_ptr() for t in grads)
    d.workspace, d.workspace_bytes = room.data_ptr(), room.numel()
    assert _lib.lib().mimk_residual_rmsnorm_bwd(ct.byref(d), T._stream()) == 0
    for g, k in zip((arrived, *grads), ("dr", "dh", "dgamma", "dpost_gamma", "dgate")):
        assert torch.equal(g, want[k]), k
