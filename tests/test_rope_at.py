"""Rotation of heads by given positions of one or several axes: against the formula in 64 bits, against what it undoes, and what is refused."""
import pytest
import torch

from zorse_b200.ops import ref
from zorse_b200.ops.api import get_ops

HALF, FP32 = 2.0 ** -8, 2.0 ** -22       # half a step of bf16; two products and a sum in fp32 (2^-24 each of |a| + |b|), twice over


def _inputs(T, heads, extra, d, sections, P, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    buf = torch.randn(T, heads * d + extra, generator=g, dtype=torch.float64).to(dtype)
    return buf, ref.rope_table(P, d, 500000.0), torch.randint(0, P, (len(sections), T), generator=g, dtype=torch.int32)


def formula64(buf, cs, positions, heads, d, sections, backward):
    h, at, out = d // 2, 0, buf.double().clone()
    size = torch.zeros_like(out)
    for axis, n in enumerate(sections):
        row = cs[positions[axis].long().clamp(0, cs.shape[0] - 1)].double()
        c, s = row[:, at:at + n], row[:, h + at:h + at + n] * (-1 if backward else 1)
        for k in range(heads):
            i = slice(k * d + at, k * d + at + n)
            j = slice(k * d + h + at, k * d + h + at + n)
            a, b = buf[:, i].double(), buf[:, j].double()
            out[:, i], out[:, j] = a * c - b * s, b * c + a * s
            size[:, i] = size[:, j] = a.abs() + b.abs()
        at += n
    return out, size


CASES = [  # T, heads, columns behind them, width, sections, rows of the table
    (1, 1, 0, 64, [32], 1), (7, 3, 64, 64, [32], 9), (255, 24, 512, 64, [32], 256), (130, 5, 128, 128, [16, 24, 24], 1000),
    (33, 4, 0, 128, [64], 70), (64, 9, 8, 32, [5, 11], 40), (19, 2, 0, 96, [13, 0, 20, 15], 131072), (50, 1, 3, 48, [24], 60),
    (21, 3, 1, 64, [20, 12], 33), (40, 2, 0, 6, [1, 2], 50), (17, 4, 0, 256, [1, 126, 1], 17), (600, 40, 1024, 128, [22, 21, 21], 5000),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("backward", [False, True])
def test_reference_by_the_formula_cpu(case, backward):
    T, heads, extra, d, sections, P = case
    buf, cs, positions = _inputs(*case, dtype=torch.float64)
    want, _ = formula64(buf, cs, positions, heads, d, sections, backward)
    assert torch.allclose(get_ops("ref").rope_at_(buf.clone(), cs, positions, heads, d, sections, backward), want, atol=1e-13)


def test_as_the_plain_rotation_cpu():
    """One axis with places that start again is the rotation of a batch of sequences."""
    ops, (buf, cs, _) = get_ops("ref"), _inputs(12, 3, 64, 64, [32], 4)
    positions = torch.arange(12, dtype=torch.int32) % 4
    assert torch.equal(ops.rope_at_(buf.clone(), cs, positions, 3, 64), ops.rope_(buf.clone(), cs, 4, 3, 64))


def test_gradient_is_the_transpose_cpu():
    ops, (buf, cs, positions) = get_ops("ref"), _inputs(9, 2, 0, 32, [10, 6], 30, dtype=torch.float64)
    dy = torch.randn(buf.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    y, dx = (ops.rope_at_(t.clone(), cs, positions, 2, 32, [10, 6], b) for t, b in ((buf, False), (dy, True)))
    assert torch.allclose((y * dy).sum(), (buf * dx).sum())


@pytest.fixture
def wrapper(monkeypatch):
    from zorse_b200.ops import sm100 as k

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_bf16", lambda t, name: None if t.dtype == torch.bfloat16 else (_ for _ in ()).throw(TypeError(name)))
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    return k


def test_refusals_cpu(wrapper):
    T, heads, d, sections = 6, 3, 64, [20, 12]
    buf, cs, positions = _inputs(T, heads, 64, d, sections, 10)
    ok = dict(buf=buf, cs=cs, positions=positions, nheads=heads, d=d, sections=sections)
    for wrong in (dict(nheads=5), dict(nheads=-1), dict(d=63), dict(sections=[20, 13]), dict(sections=[40, -8]), dict(sections=[4, 4, 4, 4, 16]),
                  dict(sections=[]), dict(sections=None), dict(positions=positions[:, :3]), dict(positions=positions.long()),
                  dict(positions=positions.t().contiguous().t()), dict(cs=cs.double()), dict(cs=cs[:0]), dict(cs=cs[:, :32].contiguous()),
                  dict(buf=buf.t().contiguous().t()), dict(buf=buf[:1].expand(T, -1)), dict(buf=buf.view(-1))):
        with pytest.raises(ValueError):
            wrapper.rope_at_(**{**ok, **wrong})
    with pytest.raises(TypeError):
        wrapper.rope_at_(**{**ok, "buf": buf.float()})


# ------------------------------------------------------------------------------------------------------------------ on the GPU
@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("backward", [False, True])
def test_kernel(ops, case, backward):
    T, heads, extra, d, sections, P = case
    buf, cs, positions = _inputs(*case)
    want, size = formula64(buf, cs, positions, heads, d, sections, backward)
    x = buf.cuda()
    got = ops.rope_at_(x, cs.cuda(), positions.cuda(), heads, d, sections, backward)
    assert got.data_ptr() == x.data_ptr() and torch.equal(got[:, heads * d:].cpu(), buf[:, heads * d:])
    assert ((got.cpu().double() - want).abs() <= HALF * want.abs() + FP32 * size)[:, :heads * d].all()


@pytest.mark.gpu
def test_strides_streams_graphs_and_positions_outside(ops):
    T, heads, d, sections = 77, 4, 64, [12, 20]
    buf, cs, positions = _inputs(T, heads, 0, d, sections, 50)
    cs, positions = cs.cuda(), positions.cuda()
    want = ops.rope_at_(buf.cuda(), cs, positions, heads, d, sections)
    for before in (8, 3):      # rows on and off a 16-byte boundary, inside a wider buffer whose other columns stay
        wide = torch.full((T, before + heads * d + 24), 7.0, dtype=torch.bfloat16, device="cuda")
        wide[:, before:before + heads * d] = buf.cuda()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.rope_at_(wide[:, before:before + heads * d], cs, positions, heads, d, sections)
        torch.cuda.current_stream().wait_stream(s)
        off = (wide[:, before:before + heads * d].float() - want.float()).abs()
        assert (off <= 2 * HALF * want.float().abs() + 2e-6).all()     # (another order of the same two roundings)
        assert (wide[:, :before] == 7).all() and (wide[:, before + heads * d:] == 7).all()
    x, src = torch.empty_like(want), buf.cuda()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x.copy_(src)
        ops.rope_at_(x, cs, positions, heads, d, sections)
    for _ in range(2):
        graph.replay()
        assert torch.equal(x, want)
    outside = torch.where(positions % 2 == 0, positions + 1000, positions - 2 ** 31)
    got = ops.rope_at_(buf.cuda(), cs, outside, heads, d, sections)
    assert torch.equal(got, ops.rope_at_(buf.cuda(), cs, outside.clamp(0, 49), heads, d, sections))
    assert ops.rope_at_(buf[:0].cuda(), cs, positions[:, :0].contiguous(), heads, d, sections).shape == (0, heads * d)
    assert torch.equal(ops.rope_at_(buf.cuda(), cs, positions, 0, d, sections).cpu(), buf)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 90])
def test_offsets_that_pass_32_bits(ops, d):
    T, heads, sections = 300000, 60 * 128 // d, [d // 4, d // 2 - d // 4]
    assert T * heads * d > 2 ** 31
    torch.manual_seed(0)
    buf = torch.randn(T, heads * d, dtype=torch.bfloat16, device="cuda")
    cs, positions = torch.randn(500, d, device="cuda"), torch.randint(0, 500, (2, T), dtype=torch.int32, device="cuda")
    near = 2 ** 31 // (heads * d)
    rows = torch.tensor([0, near - 1, near, near + 1, T - 1], device="cuda")
    want = ops.rope_at_(buf[rows], cs, positions[:, rows].contiguous(), heads, d, sections)
    assert torch.equal(ops.rope_at_(buf, cs, positions, heads, d, sections)[rows], want)
