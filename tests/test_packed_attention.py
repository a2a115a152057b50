"""Attention over packed sequences: against the formulas in 64 bits sequence by sequence, against differences, and what is refused."""
import math
import pathlib
import re

import pytest
import torch

from zorse_b200.ops import packed
from zorse_b200.ops.api import get_ops

HALF = 2.0 ** -8          # half a step of bf16, relative


def _offsets(lengths):
    return torch.tensor([0, *lengths]).cumsum(0).to(torch.int32)


def _inputs(T, Hq, Hkv, D, seed=0, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype)

    return normal(T, (Hq + 2 * Hkv) * D), normal(T, Hq * D)


def _hidden(n, causal, window, device):
    i = torch.arange(n, device=device)
    hide = torch.zeros(n, n, dtype=torch.bool, device=device)
    if causal:
        hide |= i > i[:, None]
    if window:
        hide |= i[:, None] - i >= window
    return hide


def _each(qkv, lengths, Hq, Hkv, D):
    """(slice, q [Hq, n, D], k and v for each query head) of every sequence, in 64 bits."""
    at = 0
    for n in lengths:
        x = qkv[at:at + n].double().view(n, Hq + 2 * Hkv, D).transpose(0, 1)
        k, v = (x[Hq + i * Hkv:Hq + (i + 1) * Hkv].repeat_interleave(Hq // Hkv, 0) for i in (0, 1))
        if n:
            yield slice(at, at + n), x[:Hq], k, v
        at += n


def forward64(qkv, lengths, Hq, Hkv, D, causal, window):
    """out, lse, and the size of what an output is summed from."""
    T = qkv.shape[0]
    out, size = (torch.zeros(T, Hq, D, dtype=torch.float64, device=qkv.device) for _ in range(2))
    lse = torch.full((Hq, T), -math.inf, dtype=torch.float64, device=qkv.device)
    for at, q, k, v in _each(qkv, lengths, Hq, Hkv, D):
        s = (q @ k.transpose(1, 2) / math.sqrt(D)).masked_fill(_hidden(q.shape[1], causal, window, qkv.device), -math.inf)
        lse[:, at] = torch.logsumexp(s, 2)
        p = torch.softmax(s, 2)
        out[at], size[at] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    return out.reshape(T, Hq * D), lse, size.reshape(T, Hq * D)


def backward64(do, qkv, o, lse, lengths, Hq, Hkv, D, causal, window):
    """The gradient; what bf16 factors can put it off by at most; and the size of the sums behind it, for fp32's share."""
    T, c = qkv.shape[0], D ** -0.5
    grad, off, size = (torch.zeros(T, Hq + 2 * Hkv, D, dtype=torch.float64, device=qkv.device) for _ in range(3))

    def groups(x):      # over the query heads of a key head
        return x.view(Hkv, Hq // Hkv, *x.shape[1:]).sum(1).transpose(0, 1)

    for at, q, k, v in _each(qkv, lengths, Hq, Hkv, D):
        n = q.shape[1]
        g, out = (t[at].double().view(n, Hq, D).transpose(0, 1) for t in (do, o))
        p = (q @ k.transpose(1, 2) * c - lse[:, at, None].double()).masked_fill(_hidden(n, causal, window, qkv.device), -math.inf).exp()
        dp, delta = g @ v.transpose(1, 2), (g * out).sum(2, keepdim=True)
        ds, big = p * (dp - delta), p * (g.abs() @ v.abs().transpose(1, 2) + (g * out).abs().sum(2, keepdim=True))
        pt, dst, bigt = p.transpose(1, 2), ds.transpose(1, 2), big.transpose(1, 2)
        grad[at] = torch.cat([(ds @ k).transpose(0, 1) * c, groups(dst @ q) * c, groups(pt @ g)], 1)
        off[at] = torch.cat([(ds.abs() @ k.abs()).transpose(0, 1) * c, groups(dst.abs() @ q.abs()) * c, groups(pt @ g.abs())], 1)
        size[at] = torch.cat([(big @ k.abs()).transpose(0, 1) * c, groups(bigt @ q.abs()) * c, groups(pt @ g.abs())], 1)
    return tuple(x.reshape(T, -1) for x in (grad, off, size))


CASES = [  # T, lengths, query heads, key heads, width, causal, window
    (1, [1], 1, 1, 64, True, 0), (2, [1, 1], 2, 1, 128, True, 0), (3, [], 1, 1, 64, True, 0), (5, [0, 2, 0, 0, 1, 0], 3, 3, 64, True, 0),
    (128, [128], 4, 4, 128, True, 0), (256, [127, 1, 128], 4, 2, 64, True, 0), (257, [129, 127, 1], 2, 2, 128, True, 0),
    (300, [1] * 300, 2, 1, 64, True, 0), (513, [7, 250, 3, 252, 1], 5, 1, 128, True, 0), (640, [100, 90, 0, 260], 8, 2, 64, True, 0),
    (1000, [999], 4, 4, 64, True, 0), (1290, [300, 5, 985], 8, 8, 128, True, 0), (700, [200, 300, 130], 4, 1, 128, True, 65),
    (900, [900], 8, 2, 64, True, 1), (511, [400, 111], 2, 2, 64, True, 400), (384, [384], 3, 1, 64, False, 0),
    (600, [129, 60, 127, 200], 6, 2, 128, False, 0), (1027, [50, 700, 13, 260], 4, 4, 64, False, 0), (200, [], 4, 2, 128, False, 0),
    (1500, [1400], 2, 2, 128, True, 0), (2000, [3] * 600, 4, 1, 64, False, 0),
    # heads of 64 in groups: four or two of them side by side, and the odd groups that are not
    (1, [1], 4, 1, 64, True, 0), (65, [63, 2], 4, 1, 64, True, 0), (129, [1, 64, 64], 8, 2, 64, False, 0), (1100, [1000, 77], 8, 1, 64, True, 0),
    (1031, [130, 700, 191], 4, 2, 64, True, 0), (640, [100, 90, 0, 260], 2, 1, 64, True, 37), (900, [64, 64, 500, 200], 12, 2, 64, True, 150), (520, [510], 6, 3, 64, False, 0),
    (1300, [1300], 16, 2, 64, True, 0),
]


# ------------------------------------------------------------------------------------------------------------------ on the CPU
@pytest.mark.parametrize("case", [c for c in CASES if c[0] <= 700])
def test_reference_by_the_formulas_cpu(case):
    T, lengths, Hq, Hkv, D, causal, window = case
    ops = get_ops("ref")
    qkv, do = _inputs(T, Hq, Hkv, D, dtype=torch.float64)
    pk = ops.pack_sequences(_offsets(lengths), T)
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D, causal, window)
    want, lse64, _ = forward64(qkv, lengths, Hq, Hkv, D, causal, window)
    assert torch.allclose(out, want, atol=1e-12) and torch.allclose(lse, lse64, atol=1e-12)
    grad = ops.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D, causal, window)
    assert torch.allclose(grad, backward64(do, qkv, want, lse64, lengths, Hq, Hkv, D, causal, window)[0], atol=1e-11)


def test_gradient_by_differences_cpu():
    T, lengths, Hq, Hkv, D = 9, [4, 0, 3], 4, 2, 64
    qkv, do = _inputs(T, Hq, Hkv, D, dtype=torch.float64, seed=3)

    def loss(x):
        return float((forward64(x, lengths, Hq, Hkv, D, True, 0)[0] * do).sum())

    out, lse, _ = forward64(qkv, lengths, Hq, Hkv, D, True, 0)
    grad = backward64(do, qkv, out, lse, lengths, Hq, Hkv, D, True, 0)[0]
    for i, j in [(0, 0), (1, 70), (2, 4 * 64 + 3), (3, 5 * 64 + 9), (4, 6 * 64), (6, 7 * 64 + 63), (8, 5), (5, 255)]:
        h = torch.zeros_like(qkv)
        h[i, j] = 1e-5
        assert abs((loss(qkv + h) - loss(qkv - h)) / 2e-5 - float(grad[i, j])) < 1e-7


def test_bounds_and_positions_cpu():
    pk = get_ops("ref").pack_sequences(_offsets([2, 0, 3]), 7)
    assert pk.bounds.shape == (256, 2) and pk.bounds[:8].tolist() == [[0, 2], [0, 2], [2, 5], [2, 5], [2, 5], [5, 5], [5, 5], [5, 5]]
    assert pk.positions.tolist() == [0, 1, 0, 1, 2, 0, 0]
    for wrong in ([0, 3, 2], [1, 2], [0, 9]):
        with pytest.raises(ValueError):
            get_ops("ref").pack_sequences(torch.tensor(wrong, dtype=torch.int32), 7)


def test_what_lies_behind_the_last_sequence_reaches_nobody_cpu():
    T, lengths, Hq, Hkv, D = 40, [20, 9], 2, 1, 64
    ops, (qkv, do) = get_ops("ref"), _inputs(T, Hq, Hkv, D, dtype=torch.float32)
    pk = ops.pack_sequences(_offsets(lengths), T)
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
    grad = ops.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D)
    bad = qkv.clone()
    bad[29:] = float("nan")
    out2, lse2 = ops.packed_attn_fwd(bad, pk, Hq, Hkv, D)
    assert torch.equal(out, out2) and torch.equal(lse, lse2) and (out[29:] == 0).all() and (lse[:, 29:] == -math.inf).all()
    assert torch.equal(grad, ops.packed_attn_bwd(do, bad, out, lse, pk, Hq, Hkv, D)) and (grad[29:] == 0).all()


@pytest.fixture
def wrapper(monkeypatch):
    from zorse_b200.ops import sm100 as k

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_bf16", lambda t, name: None if t.dtype == torch.bfloat16 else (_ for _ in ()).throw(TypeError(name)))
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    monkeypatch.setattr(k, "_stream", lambda: None)
    return k


def test_refusals_cpu(wrapper):
    offsets = _offsets([3, 2])
    for wrong in (offsets.long(), offsets.view(1, -1), offsets[:0], offsets.repeat(2)[::2]):
        with pytest.raises(ValueError):
            wrapper.pack_sequences(wrong, 5)
    for T in (-1, packed.MOST_TOKENS + 1):
        with pytest.raises(ValueError):
            wrapper.pack_sequences(offsets, T)
    T, Hq, Hkv, D = 6, 4, 2, 64
    qkv, do = _inputs(T, Hq, Hkv, D)
    tiles = torch.zeros(1, 8, dtype=torch.int32)
    pk = packed.PackedSequences(T, torch.zeros(256, 2, dtype=torch.int32), torch.zeros(T, dtype=torch.int32), torch.zeros(1, 12, dtype=torch.int32), tiles, tiles)
    ok = dict(qkv=qkv, pk=pk, Hq=Hq, Hkv=Hkv, D=D)
    calls = [(wrapper.packed_attn_fwd, ok, []),
             (wrapper.packed_attn_bwd, ok | dict(do=do, o=do, lse=torch.zeros(Hq, T)),
              [dict(do=do[:3]), dict(o=do[:, :64]), dict(do=do.t().contiguous().t()), dict(lse=torch.zeros(T, Hq)), dict(lse=torch.zeros(Hq, T).double())])]
    for call, good, more in calls:
        for wrong in [dict(qkv=qkv[:5]), dict(qkv=qkv.t().contiguous().t()), dict(Hkv=3), dict(Hkv=0), dict(Hq=0), dict(D=32), dict(window=-1),
                      dict(window=4, causal=False), dict(pk=packed.pack(offsets, T)), dict(pk=pk._replace(bounds=pk.bounds[:-1])),
                      dict(pk=pk._replace(order_keys=tiles.long())), dict(pk=pk._replace(order_pairs=tiles)), dict(pk=pk._replace(tokens=5))] + more:
            with pytest.raises(ValueError):
                call(**{**good, **wrong})
        with pytest.raises(TypeError):
            call(**{**good, "qkv": qkv.float()})
    with pytest.raises(ValueError):
        get_ops("ref").packed_attn_fwd(qkv, packed.pack(offsets, T), Hq, Hkv, D, False, 4)


def test_the_issuer_of_four_chains_walks_as_a_warp_cpu():
    """As in the kernels of equal sequences: every wait is the warp's, every issue is followed by a warp barrier, nothing is read ahead of chain_wait."""
    text = (pathlib.Path(__file__).resolve().parent.parent / "csrc/attn/packed_fwd_groups.cuh").read_text()
    body = text.split("const bool elected = elect_one();")[1]
    body = body[:body.index("// ----")]
    assert not re.search(r"\bmbar_wait\(", body)
    for m in re.finditer(r"if \([^()\n]*\belected\) (\{|[^\n{]*\n)", body):
        end = m.end()
        if m.group(1) == "{":
            depth = 1
            while depth:
                depth += {"{": 1, "}": -1}.get(body[end], 0)
                end += 1
        assert re.sub(r"//[^\n]*", "", body[end:]).split()[0] == "__syncwarp();"
    assert text.index("chain_wait();") < text.index("load_packed(") and not re.search(r"__ldg|ld_nc|__restrict__", text)


# ------------------------------------------------------------------------------------------------------------------ on the GPU
@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


# Scores are fp32 sums of D products of bf16 values and exponentials fp32 (2^-22 relative, and the scores' own error of 2^-20 or less of
# |q| |k| / sqrt(D) < 60): weights are within 2^-14 of themselves before they are rounded to bf16.
FP32 = 2.0 ** -14


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_bounds_and_orders(ops, case):
    T, lengths = case[:2]
    pk, want = ops.pack_sequences(_offsets(lengths).cuda(), T), packed.pack(_offsets(lengths), T)
    assert torch.equal(pk.bounds.cpu(), want.bounds) and torch.equal(pk.positions.cpu(), want.positions)
    b, total = want.bounds, sum(lengths)

    def of(row):       # the longest sequence first, then as they lie
        lo, hi = b[row].tolist()
        return lo - hi, lo

    for records, rows, keys in ((pk.order_pairs, 256, False), (pk.order_tiles, 128, False), (pk.order_keys, 128, True)):
        count = -(-T // rows)
        order = sorted(range(count), key=lambda i: (*of(max(min(rows * (i + 1), total) - 1, rows * i)), i) if keys else (*of(rows * i), -i))
        halves = [torch.tensor(order) * rows + h for h in range(0, rows, 128)]
        ends = [b[h] for h in halves] + [b[h + 127] for h in halves]           # bounds of the first rows, of the last ones; tile, total
        all_of_it = torch.cat([*ends, torch.tensor(order)[:, None], torch.full((count, 1), total)], 1)
        assert torch.equal(records[:, :all_of_it.shape[1]].cpu(), all_of_it.to(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(ops, case):
    T, lengths, Hq, Hkv, D, causal, window = case
    qkv, do = (x.cuda() for x in _inputs(T, Hq, Hkv, D))
    total = sum(lengths)
    qkv[total:], do[total:] = float("nan"), float("inf")      # of no sequence: whatever it is
    pk = ops.pack_sequences(_offsets(lengths).cuda(), T)
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D, causal, window)
    want, lse64, size = forward64(qkv, lengths, Hq, Hkv, D, causal, window)
    assert ((out.double() - want).abs() <= HALF * (size + want.abs()) + (FP32 + HALF ** 2) * size).all()
    assert torch.equal(lse.isinf(), lse64.isinf()) and ((lse.double() - lse64).abs()[:, :total] <= FP32).all()
    assert (out[total:] == 0).all()
    o, lse = want.to(torch.bfloat16), lse64.float()
    o[total:] = float("nan")
    got = ops.packed_attn_bwd(do, qkv, o, lse, pk, Hq, Hkv, D, causal, window)
    grad, off, size = backward64(do, qkv, o, lse, lengths, Hq, Hkv, D, causal, window)
    assert ((got.double() - grad).abs() <= HALF * (off + grad.abs()) + HALF ** 2 * off + FP32 * size).all()
    assert (got[total:] == 0).all()
    ops.k.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_equal_sequences_as_a_batch(ops, D):
    """Sequences of 256 tokens packed: the bits of the batch of equal sequences."""
    B, S, Hq, Hkv = 5, 256, 4, 2 if D == 128 else 4         # (heads of 64 in groups have a kernel with other tiles)
    qkv, do = (x.cuda() for x in _inputs(B * S, Hq, Hkv, D))
    pk = ops.pack_sequences(_offsets([S] * B).cuda(), B * S)
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
    out2, lse2 = ops.attn_fwd(qkv, B, S, Hq, Hkv, D)
    assert torch.equal(out, out2) and torch.equal(lse, lse2.transpose(0, 1).reshape(Hq, B * S))
    grad = ops.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D)
    grad2 = ops.attn_bwd(do, qkv, out2, lse2, B, S, Hq, Hkv, D)
    assert (grad.float() - grad2.float()).abs().max() <= 2 * HALF * grad2.float().abs().max()   # (heads of a group may be added in another order)


@pytest.mark.gpu
def test_streams_graphs_and_repeats(ops):
    T, lengths, Hq, Hkv, D = 900, [100, 500, 0, 230], 8, 2, 64
    qkv, do = (x.cuda() for x in _inputs(T, Hq, Hkv, D))
    offsets = _offsets(lengths).cuda()

    def both():
        pk = ops.pack_sequences(offsets, T)
        out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
        return out, lse, ops.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D)

    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = both()
    for lens in (lengths, [900], [3] * 300, lengths):       # other sequences in the same tokens: offsets are read by the kernels
        offsets.copy_(torch.nn.functional.pad(_offsets(lens), (0, max(0, offsets.numel() - len(lens) - 1)), value=sum(lens))[:offsets.numel()])
        graph.replay()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    assert all(torch.equal(a, b) for a, b in zip(again, first))
    ops.k.check_status()


@pytest.mark.gpu
def test_offsets_that_do_not_rise_stay_inside(ops):
    """Their results mean nothing; every token is still written, and nothing else is touched."""
    T, Hq, Hkv, D = 700, 2, 1, 64
    qkv, do = (x.cuda() for x in _inputs(T, Hq, Hkv, D))
    for wrong in ([0, 600, 100, 5000], [-50, 300, 2 ** 31 - 1], [500, 400, 300, 0], [2 ** 31 - 1, -(2 ** 31)], [0, 700, 0, 700]):
        pk = ops.pack_sequences(torch.tensor(wrong, dtype=torch.int32, device="cuda"), T)
        assert ((pk.bounds >= 0) & (pk.bounds <= T)).all()
        for order, n, at in ((pk.order_pairs, 3, 8), (pk.order_tiles, 6, 4), (pk.order_keys, 6, 4)):
            assert sorted(order[:, at].tolist()) == list(range(n))
        out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
        ops.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D)
        ops.k.check_status()


@pytest.mark.gpu
def test_no_tokens(ops):
    pk = ops.pack_sequences(torch.zeros(1, dtype=torch.int32, device="cuda"), 0)
    qkv = torch.zeros(0, 4 * 64, dtype=torch.bfloat16, device="cuda")
    out, lse = ops.packed_attn_fwd(qkv, pk, 2, 1, 64)
    assert out.shape == (0, 128) and lse.shape == (2, 0)
    assert ops.packed_attn_bwd(out, qkv, out, lse, pk, 2, 1, 64).shape == qkv.shape


@pytest.mark.gpu
def test_offsets_that_pass_32_bits(ops):
    """Rows on both sides of element 2^31 of qkv, and the last: the same bits as of their sequences alone, which lie on the same tiles.
    (Gradients of keys and values only nearly: a short batch divides a group's query heads among more CTAs, so sums go in another order.)"""
    n, count, Hq, Hkv, D = 1024, 342, 48, 1, 128
    T = n * count
    assert T * Hq * D > 2 ** 31
    torch.manual_seed(0)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda")
    do = torch.randn(T, Hq * D, dtype=torch.bfloat16, device="cuda")
    pk = ops.pack_sequences(torch.arange(count + 1, dtype=torch.int32, device="cuda") * n, T)
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
    grad = ops.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D)
    one = ops.pack_sequences(torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
    for i in (0, 2 ** 31 // qkv.shape[1] // n, count - 1):
        at = slice(i * n, i * n + n)
        o, s = ops.packed_attn_fwd(qkv[at], one, Hq, Hkv, D)
        assert torch.equal(o, out[at]) and torch.equal(s, lse[:, at])
        dq = slice(0, Hq * D)
        assert torch.equal(ops.packed_attn_bwd(do[at], qkv[at], o, s, one, Hq, Hkv, D)[:, dq], grad[at][:, dq])
        want, off, size = backward64(do[at], qkv[at], o, s, [n], Hq, Hkv, D, True, 0)
        assert ((grad[at].double() - want).abs() <= HALF * (off + want.abs()) + HALF ** 2 * off + FP32 * size).all()
    ops.k.check_status()
