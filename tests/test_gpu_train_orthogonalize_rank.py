"""The orthogonalised update of matrices with hardly any rank: rows that are nearly parallel, a few large ones among small ones, singular values of two or three sizes. What a product rounds
away of such a matrix lies in its small directions, which grow by 3.4 a step.

Tolerance, of all of them: the documented 3e-3 of the result's 2-norm before it is rounded to BF16, and that rounding, half a step of each value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
DEFAULT = (3.4445, -4.7750, 2.0315)


def matrix(kind, m, n, seed):
    """F32 [m, n], m <= n."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, dtype=torch.float64)  # noqa: E731
    name, _, much = kind.partition(" ")
    if name == "parallel":          # rows that are multiples of one, and noise
        x = normal(m, 1) @ normal(1, n) + float(much) * normal(m, n)
    elif name == "two":             # two parallel rows that outweigh all others
        x = torch.zeros(m, n, dtype=torch.float64)
        x[:2] = normal(1, n)
        x += float(much) * normal(m, n)
    else:                           # "levels": half of the singular values 1, half of them `much`
        left, right = torch.linalg.qr(normal(m, m))[0], torch.linalg.qr(normal(n, m))[0]
        values = torch.ones(m, dtype=torch.float64)
        values[(m + 1) // 2:] = float(much)
        x = (left * values) @ right.mT
    return x.float()


def exact(x, steps, eps=1e-7):
    x = x.double()
    m, n = x.shape
    x = x / (torch.linalg.matrix_norm(x) + eps)
    x = x if m <= n else x.mT
    for p, q, r in steps:
        a = x @ x.mT
        x = p * x + (q * a + r * (a @ a)) @ x
    return x if m <= n else x.mT


def half_step(t):
    """Half the distance between neighbours of each BF16 value (2^-8 of the power of two at or below it)."""
    return torch.exp2(torch.floor(torch.log2(t.double().abs().clamp(min=2.0 ** -126))) - 8)


def check(x, got, steps=(DEFAULT,) * 5, within=3e-3):
    want = exact(x, steps)
    off, rounding = (got.double() - want).norm(), half_step(got).norm()
    assert float(off) <= within * float(want.norm()) + float(rounding), (float(off / want.norm()), float(rounding / want.norm()))


# one CTA for each (wide and tall), and launches of their own for each product
SHAPES = [(1, 200), (2, 128), (2, 256), (3, 40), (8, 256), (64, 256), (128, 128), (1, 1000), (2, 300), (2, 1000), (8, 1000), (32, 1000), (128, 520), (200, 264), (256, 700), (520, 520)]
KINDS = ["parallel 1e-2", "parallel 1e-3", "parallel 1e-4", "parallel 1e-6", "two 1e-3", "two 1e-5", "levels 1e-1", "levels 1e-2", "levels 1e-3", "levels 1e-5"]


@pytest.mark.parametrize("shape", SHAPES)
def test_hardly_any_rank(shape):
    from mimir_b200 import tensor as T
    for seed, kind in enumerate(KINDS):
        x = matrix(kind, *shape, seed).cuda()
        check(x, T.orthogonalize(x))
        tall = x.t().contiguous()
        check(tall, T.orthogonalize(tall))
        half = x.to(BF16)
        check(half, T.orthogonalize(half))
    T.device_status()


@pytest.mark.parametrize("shape", [(2, 256), (16, 200), (2, 1000), (150, 300)])
def test_more_and_other_steps(shape):
    """Eight of the default steps: what is off after five of them grows at most as a singular value's change does in three, whose derivative is largest at 0, 3.4445 ^ 3. And 25 steps of
    (1.5, -0.5, 0), in which small values grow by 2.5e4: its derivative is at most 1.5 and vanishes where the values end, so that what one step leaves is gone in the next ones."""
    from mimir_b200 import tensor as T
    for seed, kind in enumerate(KINDS):
        x = matrix(kind, *shape, seed).cuda()
        check(x, T.orthogonalize(x, steps=8), (DEFAULT,) * 8, 3e-3 * DEFAULT[0] ** 3)
        check(x, T.orthogonalize(x, steps=25, coefficients=(1.5, -0.5, 0.0)), ((1.5, -0.5, 0.0),) * 25)
    T.device_status()


def test_a_matrix_comes_out_the_same_where_a_stack_has_other_tiles():
    """Alone, A's tiles are of single SMs; of many matrices they are of pairs."""
    from mimir_b200 import tensor as T
    g = torch.Generator(device="cuda").manual_seed(5)
    for shape in ((16, 1024, 4096), (16, 4096, 1024), (40, 512, 2048), (30, 300, 5000)):
        x = torch.randn(shape, generator=g, device="cuda", dtype=BF16)
        got = T.orthogonalize(x)
        for i in (0, shape[0] // 2, shape[0] - 1):
            assert torch.equal(T.orthogonalize(x[i]), got[i]), (shape, i)
    T.device_status()
