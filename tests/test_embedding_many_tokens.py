"""Embedding gradient by token, more tokens than are put in order at once: a row of the table is still read, added to and rounded once."""
import pytest
import torch

from zorse_b200.ops.api import get_ops

CHUNK = 32768


def _rows(T, H, seed=0):
    return torch.randn(T, H, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _ids(T, V, kind):
    g = torch.Generator().manual_seed(T + V)
    ids = torch.randint(0, V, (T,), generator=g)
    if kind == "one":
        ids[:] = V - 1
    elif kind == "hot":
        ids[torch.rand(T, generator=g) < 0.3] = V // 3
    elif kind == "ends":                # the lowest and the highest id, and equal ids on both sides of the chunks' borders
        ids[torch.rand(T, generator=g) < 0.2] = 0
        ids[torch.rand(T, generator=g) < 0.2] = V - 1
        for c in range(CHUNK, T, CHUNK):
            ids[c - 40:c + 40] = V // 2
    elif kind == "apart":               # each chunk has ids of its own, the later chunks the lower ones
        chunks = -(-T // CHUNK)
        ids = ids % max(V // chunks, 1) + (chunks - 1 - torch.arange(T) // CHUNK) * (V // chunks)
    return ids


def test_the_reference_rounds_once_cpu():
    table = torch.full((2, 8), 256.0, dtype=torch.bfloat16)
    ids = torch.tensor([1, 1])
    get_ops("ref").embedding_bwd(ids, torch.full((2, 8), 0.9).bfloat16(), table, by_token=True)
    assert (table[1] == 258).all() and (table[0] == 256).all()


@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [2, 3])
def test_a_bf16_row_is_rounded_once(chunks):
    """256 + 0.9 rounds to 256 in bf16 however often; 256 + 0.9 + 0.9 is 258."""
    T = chunks * CHUNK
    ids = torch.zeros(T, dtype=torch.long)
    ids[torch.arange(chunks) * CHUNK + 7] = 5
    dout = torch.zeros(T, 16)
    dout[ids == 5] = 0.9
    table = torch.full((9, 16), 256.0, dtype=torch.bfloat16, device="cuda")
    get_ops("sm100").embedding_bwd(ids.cuda(), dout.bfloat16().cuda(), table, by_token=True)
    want = torch.full((9, 16), 256.0)
    want[5] = (256 + chunks * torch.tensor(0.9).bfloat16().float()).bfloat16().float()
    assert torch.equal(table.float().cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,H", [(CHUNK + 1, 5000, 40), (2 * CHUNK, 300, 264), (2 * CHUNK + 1, 2, 8), (70001, 262145, 8), (5 * CHUNK - 3, 40000, 72),
                                   (40000, 1, 16), (33000, 32000, 1032)])
@pytest.mark.parametrize("kind", ["any", "one", "hot", "ends", "apart"])
@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
def test_sums(T, V, H, kind, grads):
    """One rounding of the sum to the table's type, and fp32 additions: at most 32 rows of a piece one behind the other, then the
    parts of a run.  Eight warps share those, four rows to a piece at the least, or one has up to 17; eight partial sums, the
    factor and the old value are the rest."""
    ops = get_ops("sm100")
    ids, dout, scale = _ids(T, V, kind), _rows(T, H), 1.3
    old = torch.randn(V, H, generator=torch.Generator().manual_seed(9)).to(grads)
    runs = []
    for _ in range(2):
        table = old.cuda()
        ops.embedding_bwd(ids.cuda(), dout.cuda(), table, scale=scale, by_token=True)
        runs.append(table.cpu())
    assert torch.equal(*runs)
    d = dout.double() * float(torch.tensor(scale))
    want = old.double().index_add(0, ids, d)
    size = old.double().abs().index_add(0, ids, d.abs())
    most = torch.bincount(ids, minlength=V).max().item()
    chain = (32 + max(17, -(-most // 4) / 8 + 1) + 10) * 2.0 ** -24
    half = torch.finfo(grads).eps / 2
    assert ((runs[0].double() - want).abs() <= half * want.abs() + (1 + half) * chain * size).all()
    unused = torch.ones(V, dtype=torch.bool)
    unused[ids] = False
    assert torch.equal(runs[0][unused], old[unused])


@pytest.mark.gpu
def test_whole_numbers_and_the_order_of_a_graph():
    """Every row is counted once, whatever chunk it lies in; a captured call gives what the eager one does."""
    ops = get_ops("sm100")
    T, V, H = 3 * CHUNK + 77, 1000, 24
    ids = _ids(T, V, "ends")
    dout = torch.randint(-3, 4, (T, H), generator=torch.Generator().manual_seed(1)).bfloat16()
    want = torch.zeros(V, H).index_add(0, ids, dout.float())
    got, a, b = torch.zeros(V, H, device="cuda"), ids.cuda(), dout.cuda()
    ops.embedding_bwd(a, b, got, by_token=True)
    assert torch.equal(got.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got.zero_()
        ops.embedding_bwd(a, b, got, by_token=True)
    for _ in range(2):
        graph.replay()
        assert torch.equal(got.cpu(), want)
