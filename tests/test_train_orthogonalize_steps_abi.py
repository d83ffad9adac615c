"""Which steps the C entry point of the orthogonalised update refuses: those whose largest singular value passes 4. And that finding it out costs a call next to nothing."""
import ctypes as C
import time

import pytest


@pytest.fixture(scope="module")
def call():
    import __graft_entry__ as entry
    entry.build()
    from mimir_b200 import _lib as lib
    L, x, kept = lib.lib(), (C.c_void_p * 1)(256), []

    def desc(*steps):
        d = lib.OrthogonalizeDesc()
        flat = [v for s in steps for v in s]
        kept.append((C.c_float * len(flat))(*flat))
        d.batch, d.m, d.n, d.x, d.out, d.coefficients, d.eps, d.scale, d.steps, d.dtype = 0, 8, 8, x, 256, kept[-1], 1e-7, 1.0, len(steps), lib.F32
        return d
    return lambda *steps: L.mimk_orthogonalize(C.byref(desc(*steps)), None), desc, L.mimk_orthogonalize


def largest(step, most):
    """Of |p v + q v^3 + r v^5| up to `most`, looked for."""
    p, q, r = step
    return max(abs(v * (p + v * v * (q + r * v * v))) for v in (most * i / 20000 for i in range(20001)))


@pytest.mark.parametrize("shape", [(1.0, 0.0, 0.0), (0.0, 1.0, 0.0), (0.0, 0.0, 1.0), (1.0, -0.5, 0.0), (3.4445, -4.775, 2.0315), (-3.4445, 4.775, -2.0315), (1.0, 0.0, -1.0), (0.0, 1.0, -1.0),
                                   (1.0, -4.0, 3.2), (1.0, 1.0, -1.5), (-0.2, -1.0, 2.0), (8.0, -23.0, 17.0)])
def test_values_up_to_4(call, shape):
    """Scaled to 2 in 1000 (of the hundredth that is kept for roundings: 1 %) below and above 4, wherever the largest value lies: at 1, between, at either root, for either sign."""
    status, _, _ = call
    by = 4 / 1.01 / largest(shape, 1.0)
    assert status(tuple(v * by * 1.002 for v in shape)) == 8
    assert status(tuple(v * by * 0.998 for v in shape)) != 8
    # of the second step, up to 1.01 times what the first leaves
    first = (0.5, 0.25, 0.0)
    by = 4 / 1.01 / largest(shape, 0.75 * 1.01)
    assert status(first, tuple(v * by * 1.002 for v in shape)) == 8
    assert status(first, tuple(v * by * 0.998 for v in shape)) != 8


def test_steps_cost_the_host_next_to_nothing(call):
    """63 steps and one that is refused: less than 2 us a step."""
    _, desc, entry = call
    d = desc(*[(3.4445, -4.775, 2.0315)] * 63, (100.0, 0.0, 0.0))
    best = 1.0
    for _ in range(50):
        start = time.perf_counter()
        assert entry(C.byref(d), None) == 8
        best = min(best, time.perf_counter() - start)
    assert best < 64 * 2e-6, best
