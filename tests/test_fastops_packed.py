"""The native calls of packed attention, rotation by positions and the Newton-Schulz products against their wrappers: the same bits, the
same number of launches, and what the native ones leave to the wrappers."""
import pytest
import torch

from zorse_b200.ops.api import get_ops
from zorse_b200.ops.ref import rope_table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    ops = get_ops("sm100")
    ops.k.status_word("cuda:0")
    return ops


def _counted(ops, call):
    before = ops.k.launch_count()
    return call(), ops.k.launch_count() - before


def _same(a, b):
    a, b = ((x,) if isinstance(x, torch.Tensor) else x for x in (a, b))
    return len(a) == len(b) and all(torch.equal(x, y) and x.dtype == y.dtype and x.shape == y.shape for x, y in zip(a, b))


@pytest.mark.parametrize("T,Hq,Hkv,D,causal,window", [(300, 4, 2, 64, True, 0), (513, 3, 3, 128, True, 100), (200, 2, 1, 64, False, 0), (260, 2, 2, 64, True, 5000)])
def test_packed_attention(ops, T, Hq, Hkv, D, causal, window):
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").bfloat16()
    do = torch.randn(T, Hq * D, generator=g, device="cuda").bfloat16()
    pk = ops.pack_sequences(torch.tensor([0, 70, 71, T - 9], dtype=torch.int32, device="cuda"), T)
    native = ops._packed_attn_fwd(qkv, pk.bounds, pk.order_pairs, pk.order_tiles, T, Hq, Hkv, D, causal, window)
    wrapped, n = _counted(ops, lambda: ops.k.packed_attn_fwd(qkv, pk, Hq, Hkv, D, causal, window))
    assert _same(native, wrapped) and n == 1
    args = do, qkv, *wrapped
    native, n = _counted(ops, lambda: ops._packed_attn_bwd(*args, pk.bounds, pk.order_tiles, pk.order_keys, T, Hq, Hkv, D, causal, window))
    wrapped, m = _counted(ops, lambda: ops.k.packed_attn_bwd(*args, pk, Hq, Hkv, D, causal, window))
    assert _same(native, wrapped) and n == m == 3
    fwd = lambda **w: ops._packed_attn_fwd(*{**dict(qkv=qkv, bounds=pk.bounds, order=pk.order_pairs, tiles=pk.order_tiles, T=T, Hq=Hq, Hkv=Hkv, D=D, causal=causal, window=window), **w}.values())  # noqa: E731
    for wrong in (dict(qkv=qkv.float()), dict(qkv=qkv[:-1]), dict(qkv=qkv.cpu()), dict(bounds=pk.bounds[:-1]), dict(order=pk.order_pairs.long()), dict(T=T + 1), dict(tiles=pk.order_pairs),
                  dict(Hkv=0), dict(D=32), dict(window=-1), dict(causal=False, window=3), dict(order=None)):
        assert fwd(**wrong) is None
    with pytest.raises(ValueError):
        ops.packed_attn_fwd(qkv[:-1], pk, Hq, Hkv, D)


@pytest.mark.parametrize("sections", [None, [32], [10, 22], [4, 8, 0, 20]])
@pytest.mark.parametrize("backward", [False, True])
def test_rope_at(ops, sections, backward):
    T, heads, d = 90, 3, 64
    buf = torch.randn(T, 5 * d, device="cuda").bfloat16()
    cs = rope_table(50, d, 1e4, "cuda")
    positions = torch.randint(0, 50, (len(sections or [1]), T), device="cuda", dtype=torch.int32)
    native, wrapped = buf.clone(), buf.clone()
    assert ops._rope_at(native, cs, positions, heads, d, sections, backward) is True
    assert torch.equal(native, ops.k.rope_at_(wrapped, cs, positions, heads, d, sections, backward)) and not torch.equal(native, buf)
    if sections is None:
        assert torch.equal(native, ops.rope_at_(buf.clone(), cs, positions[0], heads, d, sections, backward))
    for wrong in (dict(buf=buf.float()), dict(positions=positions.long()), dict(positions=positions[:, :-1]), dict(heads=6), dict(d=62), dict(sections=[31]),
                  dict(sections=[40, -8]), dict(sections=[8, 8, 8, 4, 4]), dict(cs=cs.cpu()), dict(cs=cs[:, :-2])):
        given = {**dict(buf=buf, cs=cs, positions=positions, heads=heads, d=d, sections=sections, backward=backward), **wrong}
        assert ops._rope_at(*given.values()) is None


def test_newton_schulz(ops):
    k = ops.k
    shapes = [(40, 70), (70, 40), (64, 64), (40, 70), (300, 20)]
    mats = [torch.randn(s, device="cuda").to(t) for s, t in zip(shapes, (torch.float32, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32))]
    native, n = _counted(ops, lambda: ops._orthogonalize(mats, 5, k.NEWTON_SCHULZ, k.NEWTON_SCHULZ_BYTES))
    wrapped, m = _counted(ops, lambda: k.orthogonalize(mats, 5))
    assert _same(native, wrapped) and n == m == 18
    for wrong in ([], mats + [mats[0].t()], mats + [mats[0].half()], mats + [mats[0].cpu()], mats + [torch.zeros(0, 3, device="cuda")], tuple(mats)):
        assert ops._orthogonalize(wrong, 5, k.NEWTON_SCHULZ, k.NEWTON_SCHULZ_BYTES) is None
    assert ops._orthogonalize(mats, 0, k.NEWTON_SCHULZ, k.NEWTON_SCHULZ_BYTES) is None
    p, mom = ([torch.randn(s, device="cuda") for s in shapes] for _ in range(2))
    copies = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") if i else None for i, s in enumerate(shapes)]

    def state():
        return [[x if x is None else x.clone() for x in t] for t in (p, mom, mats, copies)]

    a, b = state(), state()
    (_, n), (_, m) = (_counted(ops, lambda: ops._muon_step(*a, 0.1, 0.9, 0.2, True, 5, 0.5, k.NEWTON_SCHULZ, k.NEWTON_SCHULZ_BYTES)),
                      _counted(ops, lambda: k.muon_step(*b, lr=0.1, momentum=0.9, weight_decay=0.2, grad_scale=0.5)))
    assert n == m == 18 and all(_same([x for x in s if x is not None], [x for x in t if x is not None]) for s, t in zip(a, b))

    def declined(p, m, g, p16, momentum=0.9, iterations=5):
        return ops._muon_step(p, m, g, p16, 0.1, momentum, 0.2, True, iterations, 0.5, k.NEWTON_SCHULZ, k.NEWTON_SCHULZ_BYTES) is None

    u, v, w, y = torch.zeros(6, 4, device="cuda"), torch.zeros(6, 4, device="cuda"), torch.zeros(6, 4, device="cuda"), torch.zeros(6, 4, dtype=torch.bfloat16, device="cuda")
    for wrong in (([u], [u], [w], [y]), ([u], [v], [u], [y]), ([u], [v], [v], [y]), ([u, u], [v, w], [y, y], [None, None]), ([u], [v[:3]], [w], [y]), ([y], [v], [w], [y]),
                  ([u], [v], [w.t()], [y]), ([u], [v], [w], [u]), ([u], [v], [w.cpu()], [y]), ([u], [v], [w], [])):
        assert declined(*wrong)
        with pytest.raises(ValueError):
            ops.muon_step(*wrong, lr=0.1)
    assert declined([u], [v], [w], [y], momentum=1.0) and declined([u], [v], [w], [y], iterations=101)
