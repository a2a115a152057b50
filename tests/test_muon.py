"""Updates orthogonalised by Newton-Schulz products and Muon's step: against the formulas in 64 bits, and what is refused."""
import math
import pathlib
import re

import pytest
import torch

from zorse_b200.ops import muon
from zorse_b200.ops.api import get_ops

HALF = 2.0 ** -8            # half a step of bf16, relative


def _matrices(shapes, seed=0, dtype=torch.float32, size=1e-3):
    g = torch.Generator().manual_seed(seed)
    out = []
    for r, c in shapes:
        k = min(4, r, c)
        strong = torch.randn(r, k, generator=g) @ torch.randn(k, c, generator=g)
        out.append(((strong + torch.randn(r, c, generator=g)) * torch.randn(r, 1, generator=g).exp() * size).to(dtype))
    return out


def svd64(u, iterations=5):
    """The polynomial on the singular values themselves."""
    u = u.double()
    if not u.any():
        return torch.zeros_like(u)
    left, s, right = torch.linalg.svd(u, full_matrices=False)
    s = s / s.square().sum().sqrt()
    a, b, c = muon.COEFFICIENTS
    for _ in range(iterations):
        s = a * s + b * s ** 3 + c * s ** 5
    return left * s @ right


SHAPES = [[(1, 1)], [(1, 7), (7, 1), (2, 2)], [(64, 64)], [(63, 65), (65, 63)], [(33, 300)] * 3, [(300, 33)] * 2 + [(33, 300)], [(256, 256)] * 2,
          [(257, 255)], [(512, 700), (129, 129), (512, 700)], [(1000, 333), (333, 1000)], [(8 + 3 * i, 40 + 5 * i) for i in range(11)], [(16, 2050)],
          [(31, 17)] * 70, [(800, 801)], [(1025, 513), (513, 1030)], [(300, 5000)], [(20, 9000), (9000, 20)], [(700, 2500), (40, 40), (90, 4100)],
          [(1536, 1600)] * 4, [(100 + i, 300) for i in range(9)]]


@pytest.mark.parametrize("shapes", [s for s in SHAPES if s[0][0] * s[0][1] < 200000])
def test_reference_by_the_singular_values_cpu(shapes):
    mats = _matrices(shapes)
    for u, x in zip(mats, get_ops("ref").orthogonalize([u.double() for u in mats])):
        assert torch.allclose(x, svd64(u), atol=1e-9)


def test_reference_step_cpu():
    ops, shapes = get_ops("ref"), [(12, 20), (20, 12), (9, 9)]
    p, m, g = ([x.double() for x in _matrices(shapes, seed, size=z)] for seed, z in ((1, 0.02), (2, 4e-3), (3, 1e-3)))
    for nesterov in (True, False):
        q, w = [x.clone() for x in p], [x.clone() for x in m]
        copies = [torch.zeros(x.shape, dtype=torch.bfloat16) for x in p]
        ops.muon_step(q, w, g, copies[:2] + [None], lr=0.1, momentum=0.9, weight_decay=0.5, nesterov=nesterov, grad_scale=0.25)
        for x, mom, d, y, v, c in zip(p, m, g, q, w, copies):
            new = 0.9 * mom + 0.25 * d
            step = svd64(0.25 * d + 0.9 * new if nesterov else new) * 0.1 * 0.2 * math.sqrt(max(x.shape))
            assert torch.allclose(v, new, rtol=1e-12) and torch.allclose(y, x * 0.95 - step, atol=1e-9)
        assert torch.equal(copies[0], q[0].bfloat16()) and not copies[2].any()
    z = torch.zeros(5, 3)
    assert not ops.orthogonalize([z])[0].any()


@pytest.fixture
def wrapper(monkeypatch):
    from zorse_b200.ops import sm100 as k

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    monkeypatch.setattr(k, "_stream", lambda: None)
    return k


def test_refusals_cpu(wrapper):
    u = torch.zeros(6, 4)
    for wrong in ([u.view(-1)], [u.t()], [u, u.double()], [u.half()], [u.view(2, 3, 4)], [u.to("meta")]):
        with pytest.raises(ValueError):
            wrapper.orthogonalize([u] + wrong)
    for iterations in (0, -1, 101, 2.0):
        with pytest.raises(ValueError):
            wrapper.orthogonalize([u], iterations)
    assert wrapper.orthogonalize([]) == []
    p, m, g, y = u.clone(), u.clone(), u.clone(), u.bfloat16()
    ok = dict(p=[p], m=[m], g=[g], p16=[y], lr=1e-3)
    both = torch.zeros(12, 4)
    for wrong in (dict(p=[p, p]), dict(p=[p.bfloat16()]), dict(p=[p.t()]), dict(m=[m[:3]]), dict(m=[m.bfloat16()]), dict(g=[g.half()]), dict(g=[g.t().contiguous()]),
                  dict(p16=[u]), dict(p16=[y[:, :2]]), dict(momentum=1.0), dict(momentum=-0.1), dict(m=[p]), dict(g=[p]), dict(g=[m]),
                  dict(p=[both[:6]], m=[both[3:9]]), dict(iterations=0), dict(p=[p, p], m=[m, g], g=[y, y], p16=[None, None])):
        with pytest.raises(ValueError):
            wrapper.muon_step(**{**ok, **wrong})
    wrapper.muon_step([], [], [], [], lr=1.0)


def test_the_products_end_as_the_pair_kernel_does_cpu():
    """The loops that a warp walks together wait and issue together; the producers wait for the last release of their stages and the issuer
    for the last one of the accumulators, so the closing cluster barrier need not order memory; nothing is read before chain_wait."""
    text = (pathlib.Path(__file__).resolve().parent.parent / "csrc/optim/newton_schulz.cuh").read_text()
    producer, issuer = text.split("const bool elected = elect_one();")[1:]
    issuer = issuer[:issuer.index("// ----")]
    for body in (producer[:producer.index("// ----")], issuer):
        assert not re.search(r"\bmbar_wait\(", body)
        for m in re.finditer(r"if \([^()\n]*\belected\) (\{|[^\n{]*\n)", body):
            end = m.end()
            if m.group(1) == "{":
                depth = 1
                while depth:
                    depth += {"{": 1, "}": -1}.get(body[end], 0)
                    end += 1
            assert re.sub(r"//[^\n]*", "", body[end:]).split()[0] == "__syncwarp();"
    assert re.search(r"for \(int i = 0; i < STAGES && ok; \+\+i\) \{\s*ok = mbar_wait_warp\(&empty\[stage\], phase \^ 1, ", producer)
    assert re.search(r"for \(int i = 0; i < 2 && ok; \+\+i, \+\+local\)\s*ok = mbar_wait_warp\(&tmem_empty\[local & 1\], ",
                     issuer[issuer.rindex("umma_commit_pair(&tmem_full[buf])"):])
    assert re.search(r"chain_wait\(\);\s*chain_trigger\(\);", text) and not re.search(r"__ldg|ld_nc|__restrict__", text)


# ------------------------------------------------------------------------------------------------------------------ on the GPU
@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


# An iteration rounds X, A and B to fp16: relative to their 2-norms at most 2^-11 each, as errors of random sign 2^-11 / sqrt 3 or less, and in
# the iterations' result |a| + 3 |b| s^2 + 5 |c| s^4 stands against them by less than 3.5 + 3 x 4.8 + 5 x 2.1 (s = 1); with their signs a
# change of s goes on with a + 3 b s^2 + 5 c s^4, between -1.6 and 3.5, and near s = 1 below 0.8.  The error of A enters X through
# |b + 2 c s^2| < 1 near s = 1, that of B through 1, that of X whole, each in Frobenius norm against that of X: with two iterations' worth
# kept, sqrt(3) x 2^-11 / sqrt 3 x (1 + 0.8 + 0.64 + ...) < 5 x 2^-11.  Small singular values grow by 3.5 an iteration, errors along with them:
# another factor of 2 for matrices of which most are small.
FROBENIUS = 10 * 2.0 ** -11


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize(ops, shapes, dtype):
    mats = _matrices(shapes, dtype=dtype)
    mine = [u.cuda() for u in mats]
    got = ops.orthogonalize(mine)
    for u, v, x in zip(mats, mine, got):
        assert x.dtype == torch.bfloat16 and x.shape == u.shape and torch.equal(v.cpu(), u)
        want = svd64(u)
        off = (x.cpu().double() - want).norm() / want.norm()
        assert off <= FROBENIUS + HALF, (u.shape, off)
    ops.k.check_status()


@pytest.mark.gpu
def test_scale_does_not_matter_and_zeros_stay(ops):
    """Of any size that fp32 holds; a matrix of zeros, one entry, one direction, and NaN, which stays in its matrix."""
    u = _matrices([(130, 70)])[0].cuda()
    want = ops.orthogonalize([u])[0]
    for size in (2.0 ** 90, 2.0 ** -90):
        assert torch.equal(ops.orthogonalize([u * size])[0], want)
    one, flat = torch.zeros(130, 70, device="cuda"), torch.ones(130, 70, device="cuda")
    one[129, 3] = -5.0
    bad = u.clone()
    bad[5, 5] = float("nan")
    zero, x, y, z, again = ops.orthogonalize([torch.zeros_like(u), one, flat, bad, u])
    assert not zero.any() and z.isnan().any() and torch.equal(again, want)
    s = 1.0
    for _ in range(5):
        s = sum(k * s ** e for k, e in zip(muon.COEFFICIENTS, (1, 3, 5)))
    assert abs(float(x[129, 3]) + s) <= s * (FROBENIUS + HALF) and int(x.count_nonzero()) == 1
    assert (y.float() - s / math.sqrt(130 * 70)).abs().max() <= (FROBENIUS + HALF) * s / math.sqrt(130 * 70)


@pytest.mark.gpu
@pytest.mark.parametrize("iterations", [1, 2, 6])
def test_other_iterations(ops, iterations):
    u = _matrices([(200, 150)])[0]
    want = svd64(u, iterations)
    assert (ops.orthogonalize([u.cuda()], iterations)[0].cpu().double() - want).norm() <= (FROBENIUS + HALF) * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("reduce", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(ops, shapes, reduce, nesterov):
    p, m, g = (_matrices(shapes, seed, size=z) for seed, z in ((1, 0.02), (2, 4e-3), (3, 1e-3)))
    g = [x.to(reduce) for x in g]
    q, w, d = ([x.cuda() for x in t] for t in (p, m, g))
    copies = [torch.zeros(x.shape, dtype=torch.bfloat16, device="cuda") if i % 3 != 2 else None for i, x in enumerate(p)]
    h = dict(lr=0.02, momentum=0.9, weight_decay=0.1, nesterov=nesterov, grad_scale=0.25)
    ops.muon_step(q, w, d, copies, **h)
    for x, mom, grad, y, v, c in zip(p, m, g, q, w, copies):
        grad = grad.double() * 0.25
        new = 0.9 * mom.double() + grad
        # one fma on a factor that fp32 holds to 2^-24
        assert ((v.cpu().double() - new).abs() <= 2.0 ** -23 * (new.abs() + mom.double().abs())).all()
        step = svd64(grad + 0.9 * new if nesterov else new) * 0.02 * 0.2 * math.sqrt(max(x.shape))
        off = (y.cpu().double() - (x.double() * (1 - 0.002) - step)).norm()
        assert off <= FROBENIUS * step.norm() + 2.0 ** -22 * x.double().norm()
        assert c is None or torch.equal(c, y.bfloat16())
    ops.k.check_status()


@pytest.mark.gpu
def test_alignment_streams_graphs_and_repeats(ops):
    """Matrices off their 16-byte boundaries; another stream; the same bits twice and in a captured graph; a list cut into several."""
    shapes = [(96, 200), (200, 96), (130, 64)]
    g = [x.cuda() for x in _matrices(shapes)]
    want = ops.orthogonalize(g)
    assert all(torch.equal(a, b) for a, b in zip(want, ops.orthogonalize(g)))
    odd = []
    for x in g:
        room = torch.empty(x.numel() + 1, device="cuda")
        odd.append(room[1:].view(x.shape))
        odd[-1].copy_(x)
    for a, b in zip(want, ops.orthogonalize(odd)):
        assert (a.float() - b.float()).norm() <= (2 * FROBENIUS + HALF) * a.float().norm()     # sums of squares in another order
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = ops.orthogonalize(g)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, captured))
    old, ops.k.NEWTON_SCHULZ_BYTES = ops.k.NEWTON_SCHULZ_BYTES, 1
    try:
        cut = ops.orthogonalize(g)
    finally:
        ops.k.NEWTON_SCHULZ_BYTES = old
    assert all(torch.equal(a, b) for a, b in zip(want, cut))
    before = ops.k.launch_count()
    ops.orthogonalize(g)
    assert ops.k.launch_count() - before == 3 + 15
    empty = torch.zeros(0, 5, device="cuda")
    assert ops.orthogonalize([empty, g[0]])[0].shape == (0, 5)
    ops.muon_step([empty], [empty.clone()], [empty.clone()], [None], lr=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
def test_offsets_that_pass_32_bits(ops, turned):
    """16 entries, each the only one of its row and column, the last of all among them: one iteration takes each by its polynomial."""
    n, m = 40000, 53999
    shape = (m, n) if turned else (n, m)
    assert n * m > 2 ** 31
    u = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    rows, cols = (torch.linspace(3, size - 1, 16, device="cuda").long() for size in shape)
    u[rows, cols] = 2.0
    a, b, c = muon.COEFFICIENTS
    s = 1 / 4                # 2 / ||U||
    got = ops.orthogonalize([u], 1)[0]
    want = a * s + b * s ** 3 + c * s ** 5
    assert ((got[rows, cols].double() - want).abs() <= (FROBENIUS + HALF) * want).all()
    assert int((got != 0).sum()) == 16
    ops.k.check_status()
