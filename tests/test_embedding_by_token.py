"""Scaled token embedding and its gradient summed by token: against 64 bits, the same bits on each run, and what is refused."""
import math

import pytest
import torch

from zorse_b200.ops.api import get_ops


def _normal(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def _ids(T, V, kind, seed=3):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (T,), generator=g)
    if kind == "one":
        ids[:] = V // 2
    elif kind == "hot":
        ids[torch.rand(T, generator=g) < 0.6] = V - 1
    elif kind == "few":
        ids = ids % 5 % V
    elif kind == "runs":
        ids = ids.sort(descending=True).values
    return ids


def _bwd64(ids, dout, gtable, gpos, S, off, scale):
    """Both gradients in 64 bits, and the sizes of what is added up."""
    d = dout.double()
    g = gtable.double().index_add(0, ids, d * scale)
    ga = gtable.double().abs().index_add(0, ids, (d * scale).abs())
    if gpos is None:
        return g, ga, None, None
    at = torch.arange(ids.numel()) % S + off
    return g, ga, gpos.double().index_add(0, at, d), gpos.double().abs().index_add(0, at, d.abs())


def test_reference_backend_cpu():
    ops = get_ops("ref")
    ids, table, pos = _ids(14, 9, "few"), _normal(9, 16, dtype=torch.float32), _normal(9, 16, seed=1, dtype=torch.float32)
    y = ops.embedding_fwd(ids, table, pos, 7, 2, scale=3.0)
    want = table[ids].double() * 3 + pos.double()[torch.arange(14) % 7 + 2]
    assert torch.allclose(y.double(), want, rtol=1e-6, atol=1e-6)
    dout, gt, gp = _normal(14, 16, seed=2, dtype=torch.float32), torch.ones(9, 16), torch.ones(9, 16)
    g, _, p, _ = _bwd64(ids, dout, gt, gp, 7, 2, 3.0)
    ops.embedding_bwd(ids, dout, gt, gp, 7, 2, scale=3.0, by_token=True)
    assert torch.allclose(gt.double(), g, rtol=1e-5, atol=1e-5) and torch.allclose(gp.double(), p, rtol=1e-5, atol=1e-5)


def test_refusals_cpu(monkeypatch):
    from zorse_b200.ops import sm100 as k

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_bf16", lambda t, name: None)
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    ids, table, dout = _ids(6, 10, "any"), _normal(10, 16), _normal(6, 16)
    for args in ((ids.int(), table), (ids.repeat(2)[::2], table), (ids, table.t()), (ids, table, _normal(3, 16), 6, 0),
                 (ids, table, _normal(8, 16), 6, 3), (ids, table, _normal(8, 8), 6, 0), (ids, table, _normal(8, 16), 0, 0),
                 (ids, table, _normal(8, 16), 6, -1), (ids, table[:0])):
        with pytest.raises(ValueError):
            k.embedding_scaled(*args, scale=2.0)
    for args in ((ids, dout[:5], table), (ids, dout.t().contiguous().t(), table), (ids, dout, table.double()),
                 (ids, dout, table.float(), _normal(8, 16), 6, 0), (ids, dout, table[:0])):
        with pytest.raises(ValueError):
            k.embedding_by_token(*args)


# ---------------------------------------------------------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


@pytest.mark.gpu
@pytest.mark.parametrize("T,S,V,H,off", [(1, 1, 1, 8, 0), (7, 7, 50, 64, 2), (254, 127, 1024, 256, 0), (1000, 100, 32000, 520, 0)])
@pytest.mark.parametrize("positions", [True, False])
def test_forward(ops, T, S, V, H, off, positions):
    ids, table, pos = _ids(T, V, "any"), _normal(V, H), _normal(S + off, H, seed=1) if positions else None
    scale = math.sqrt(H)
    y = ops.embedding_fwd(ids.cuda(), table.cuda(), None if pos is None else pos.cuda(), S, off, scale=scale).cpu().double()
    a = table[ids].double() * scale
    b = pos.double()[torch.arange(T) % S + off] if positions else torch.zeros_like(a)
    # one rounding to bf16; the factor, the product and the sum in fp32
    assert ((y - a - b).abs() <= 2.0 ** -8 * (a + b).abs() + 2.0 ** -22 * (a.abs() + b.abs())).all()


SHAPES = [  # T, S, V, H
    (1, 1, 1, 8), (2, 2, 3, 64), (5, 9, 40, 64), (5, 5, 1000, 256), (3000, 4000, 700, 40), (33, 33, 7, 264), (256, 128, 32000, 512), (1000, 500, 600, 128),
    (1025, 205, 129, 72), (3000, 1000, 50257, 768), (9000, 4500, 128256, 64), (20000, 20000, 300, 32),
    (16500, 5500, 3000, 1032), (32000, 8000, 5000, 1032), (32768, 4096, 4096, 16), (32769, 32769, 70000, 24), (70001, 70001, 262145, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,S,V,H", SHAPES)
@pytest.mark.parametrize("kind", ["any", "one", "hot", "few", "runs"])
@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
def test_backward(ops, T, S, V, H, kind, grads):
    ids, dout = _ids(T, V, kind), _normal(T, H)
    gt, gp = _normal(V, H, seed=1, dtype=grads), _normal(S + 1, H, seed=2, dtype=grads)
    scale = 1.7
    g, ga, p, pa = _bwd64(ids, dout, gt, gp, S, 1, scale)
    runs = []
    for _ in range(2):
        a, b = gt.cuda(), gp.cuda()
        ops.embedding_bwd(ids.cuda(), dout.cuda(), a, b, S, 1, scale=scale, by_token=True)
        runs.append((a.cpu(), b.cpu()))
    assert all(torch.equal(x, y) for x, y in zip(*runs))
    # chunks of 32768 tokens each round their sum to the table's type; a sum's longest chain of fp32 additions has at most
    # 64 rows of a piece and a stretch of the pieces behind each other
    chunks = -(-T // 32768)
    half = torch.finfo(grads).eps / 2
    chain = (64 + T / 16) * 2.0 ** -24
    assert ((runs[0][0].double() - g).abs() <= chunks * half * ga + chain * ga).all()
    rows = -(-T // S)
    assert ((runs[0][1].double() - p).abs() <= half * p.abs() + (rows + 2) * 2.0 ** -24 * pa).all()
    unused = torch.ones(V, dtype=torch.bool)
    unused[ids] = False
    assert torch.equal(runs[0][0][unused], gt[unused])


@pytest.mark.gpu
def test_small_sums_are_exact(ops):
    """Whole numbers add up exactly in fp32, whatever the order: every row must be counted once."""
    for T, V, H in ((5000, 37, 128), (40000, 1000, 40), (16384, 3, 512)):
        ids = _ids(T, V, "hot")
        dout = torch.randint(-3, 4, (T, H), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        got = torch.zeros(V, H, device="cuda")
        ops.embedding_bwd(ids.cuda(), dout.cuda(), got, by_token=True)
        assert torch.equal(got.cpu(), torch.zeros(V, H).index_add(0, ids, dout.float()))


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,H", [(20000, 500, 64), (700, 300, 256), (4000, 9000, 520)])
@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
def test_calls_that_follow_at_once(ops, T, V, H, grads):
    """Microbatches into one table, each call begun under the end of the one before: whole numbers small enough to be exact."""
    table, want, calls = torch.zeros(V, H, dtype=grads, device="cuda"), torch.zeros(V, H), []
    for i in range(6):
        ids = _ids(T, V, ("any", "runs", "few")[i % 3], seed=i)
        dout = (torch.rand(T, H, generator=torch.Generator().manual_seed(i)) < 0.002).to(torch.bfloat16)
        want.index_add_(0, ids, dout.float())
        calls.append((ids.cuda(), dout.cuda()))
    assert want.max() <= 256
    for ids, dout in calls:
        ops.embedding_bwd(ids, dout, table, by_token=True)
    assert torch.equal(table.float().cpu(), want)


@pytest.mark.gpu
def test_ids_outside_the_table_count_as_the_nearest(ops):
    V, H = 11, 32
    ids = torch.tensor([-5, 0, 10, 11, 2 ** 40, -2 ** 40, 3])
    inside = ids.clamp(0, V - 1)
    table, dout = _normal(V, H).cuda(), _normal(7, H).cuda()
    assert torch.equal(ops.embedding_fwd(ids.cuda(), table, scale=2.0), ops.embedding_fwd(inside.cuda(), table, scale=2.0))
    a, b = torch.zeros(V, H, device="cuda"), torch.zeros(V, H, device="cuda")
    ops.embedding_bwd(ids.cuda(), dout, a, by_token=True)
    ops.embedding_bwd(inside.cuda(), dout, b, by_token=True)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_no_tokens_and_a_captured_graph(ops):
    V, H, T = 50, 64, 900
    table = torch.ones(V, H, device="cuda")
    ops.embedding_bwd(torch.empty(0, dtype=torch.long, device="cuda"), torch.empty(0, H, dtype=torch.bfloat16, device="cuda"), table,
                      by_token=True)
    assert (table == 1).all()
    assert ops.embedding_fwd(torch.empty(0, dtype=torch.long, device="cuda"), table.bfloat16(), scale=2.0).shape == (0, H)
    ids, dout = _ids(T, V, "hot").cuda(), _normal(T, H).cuda()
    want = torch.zeros(V, H, device="cuda")
    ops.embedding_bwd(ids, dout, want, scale=2.0)
    got = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got.zero_()
        ops.embedding_bwd(ids, dout, got, scale=2.0)
    for _ in range(2):
        graph.replay()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_refused_by_the_library(ops):
    from zorse_b200.ops.sm100 import KernelError

    ids = torch.zeros(4, dtype=torch.long, device="cuda")
    with pytest.raises(KernelError):
        ops.embedding_fwd(ids, torch.zeros(5, 12, dtype=torch.bfloat16, device="cuda"), scale=2.0)
    with pytest.raises(KernelError):
        ops.embedding_bwd(ids, torch.zeros(4, 0, dtype=torch.bfloat16, device="cuda"), torch.zeros(5, 0, device="cuda"), by_token=True)
    dout = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros(1 + 5 * 16, device="cuda")[1:].view(5, 16)
    with pytest.raises(KernelError):
        ops.embedding_bwd(ids, dout, off, by_token=True)
