"""Newton-Schulz products on matrices whose singular values fall: of low rank, by a power, blocks of zeros.  Against the polynomial on the
singular values in 64 bits; what the rounding of X leaves where a matrix has nothing grows by 3.4 an iteration."""
import math

import pytest
import torch

from zorse_b200.ops import muon
from zorse_b200.ops.api import get_ops

A, B, C = muon.COEFFICIENTS


def _matrix(kind, rows, cols, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = min(rows, cols)
    if kind == "zero rows":
        u = torch.zeros(rows, cols)
        u[::9] = torch.randn(u[::9].shape, generator=g)
        return u
    if kind[0] == "r":
        r = int(kind[1:])
        return torch.randn(rows, r, generator=g) @ torch.randn(r, cols, generator=g)
    left, right = (torch.linalg.qr(torch.randn(size, n, generator=g, dtype=torch.float64))[0] for size in (rows, cols))
    return (left * torch.arange(1, n + 1, dtype=torch.float64) ** -float(kind[1:]) @ right.t()).float()


def exact_and_bound(u, iterations=5):
    """The result in 64 bits, and how far off the products may be, as a share of its norm."""
    left, s, right = torch.linalg.svd(u.double(), full_matrices=False)
    s = s / s.norm()
    norms = [float(s.norm())]
    for _ in range(iterations):
        s = A * s + B * s ** 3 + C * s ** 5
        norms.append(float(s.norm()))
    # Every X is rounded: 11 bits in fp16, 19 with its remainder (all iterations but the last two, and the result), so errors of 2^-11 or 2^-19
    # of a value at most, of random sign 1 / sqrt 3 of that in root mean square.  Where X has nothing they grow by A an iteration.
    off = [A ** (iterations - k) * norms[k] * (2.0 ** -11 if k + 2 >= iterations else 2.0 ** -19) for k in range(iterations + 1)]
    # Where X has something, the products see it without its remainder, which is off by the remainder times A - f' < 5.2 (f the polynomial, f' > -1.7)
    # and shrinks by 0.8 an iteration near 1; A and B are rounded as tests/test_muon.py counts it (5 times 2^-11, sqrt 3 within).
    off += [5.2 * 2.0 ** -11 * (1 + 0.8 + 0.64) * max(norms), 5 * math.sqrt(3) * 2.0 ** -11 * max(norms)]
    return left * s @ right, math.sqrt(sum(x * x for x in off) / 3) / norms[-1]


KINDS = ["r1", "r4", "r16", "r64", "r256", "k0.5", "k1", "k1.5", "k2", "k4", "zero rows"]
SHAPES = [(512, 768), (300, 1000), (1000, 300), (1024, 1024)]


@pytest.mark.parametrize("kind", KINDS)
def test_reference_cpu(kind):
    u = _matrix(kind, 96, 130).double()
    assert torch.allclose(get_ops("ref").orthogonalize([u])[0], exact_and_bound(u)[0], atol=1e-8)


@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(ops, shape):
    mats = [_matrix(kind, *shape, seed=i) for i, kind in enumerate(KINDS)]
    for kind, u, got in zip(KINDS, mats, ops.orthogonalize([u.cuda() for u in mats])):
        want, bound = exact_and_bound(u)
        off = float((got.cpu().double() - want).norm() / want.norm())
        assert off <= math.hypot(bound, 2.0 ** -8 / math.sqrt(3)), (kind, off, bound)      # (and the result's own rounding to bf16)
    ops.k.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("iterations", [1, 2, 3, 4, 7])
def test_other_iterations(ops, iterations):
    mats = [_matrix(kind, 260, 400, seed=i) for i, kind in enumerate(KINDS)]
    for kind, u, got in zip(KINDS, mats, ops.orthogonalize([u.cuda() for u in mats], iterations)):
        want, bound = exact_and_bound(u, iterations)
        off = float((got.cpu().double() - want).norm() / want.norm())
        assert off <= math.hypot(bound, 2.0 ** -8 / math.sqrt(3)), (kind, off, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_muon_step(ops, shape):
    """The step alone: weights of zeros without decay become minus the step, in fp32."""
    mats = [_matrix(kind, *shape, seed=i) for i, kind in enumerate(KINDS)]
    p, m = ([torch.zeros(shape, device="cuda") for _ in mats] for _ in range(2))
    ops.muon_step(p, m, [u.cuda() for u in mats], [None] * len(mats), lr=1.0, momentum=0.9, grad_scale=0.5)
    for kind, u, got in zip(KINDS, mats, p):
        want, bound = exact_and_bound(u)
        want = want * -muon.SCALE * math.sqrt(max(shape))
        off = float((got.cpu().double() - want).norm() / want.norm())
        assert off <= bound, (kind, off, bound)
    ops.k.check_status()


@pytest.mark.gpu
def test_many_shapes_side_by_side(ops):
    """Of each matrix the bits that it has alone: remainders lie in the workspace one behind the other."""
    shapes = [(33, 70), (70, 33), (64, 64), (31, 65), (257, 130), (5, 700), (33, 70), (1, 3), (96, 1030), (40, 40), (65, 63)]
    mats = [_matrix("r1", *s, seed=i).cuda() for i, s in enumerate(shapes)]
    assert all(torch.equal(x, ops.orthogonalize([u])[0]) for u, x in zip(mats, ops.orthogonalize(mats)))


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
def test_remainders_that_pass_32_bits(ops, turned):
    """A block of rank 1 at the far corner of a matrix of more than 2^31 elements: as exact as by itself."""
    n, m, k = 40000, 53999, 300
    shape = (m, n) if turned else (n, m)
    assert n * m > 2 ** 31
    block = _matrix("r1", k, k).bfloat16()
    u = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    u[-k:, -k:] = block.cuda()
    got = ops.orthogonalize([u])[0]
    want, bound = exact_and_bound(block.float())
    off = float((got[-k:, -k:].cpu().double() - want).norm() / want.norm())
    assert off <= math.hypot(bound, 2.0 ** -8 / math.sqrt(3)), (off, bound)
    assert int(got.count_nonzero()) == int(got[-k:, -k:].count_nonzero())
    ops.k.check_status()
