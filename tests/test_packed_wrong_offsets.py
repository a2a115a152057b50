"""Packings that do not rise from 0 to at most T: refused where their values can be seen, and NaN throughout where they cannot."""
import pytest
import torch

from zorse_b200.ops import packed
from zorse_b200.ops.api import get_ops

T = 700
MANY = list(range(0, 15 * packed.PACK_SCAN, 5))          # more sequences than a block of the plan looks at for itself
WRONG = [  # offsets, tokens
    ([10, 300, 700], T), ([0, 600, 100, 700], T), ([0, 300, 701], T), ([0, 300, 2 ** 31 - 1], T), ([-1, 300, 700], T), ([5], T), ([-7], T),
    ([0, 300, 299, 299, 700], T), ([0] * 500 + [1, 0] + [700] * 500, T),
    (MANY[:9000] + [MANY[9000] - 6] + MANY[9001:], MANY[-1]), (MANY + [MANY[-1] - 1], MANY[-1]), (MANY, MANY[-1] - 1), ([1] + MANY[1:], MANY[-1]),
]
HEADS = [(4, 1, 64), (4, 2, 64), (2, 2, 64), (6, 3, 64), (8, 1, 128), (2, 2, 128)]


@pytest.mark.parametrize("offsets,tokens", WRONG)
def test_the_reference_refuses_cpu(offsets, tokens):
    with pytest.raises(ValueError):
        get_ops("ref").pack_sequences(torch.tensor(offsets, dtype=torch.int32), tokens)


@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


def _inputs(tokens, Hq, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    return (torch.randn(tokens, n * D, generator=g, device="cuda").bfloat16() for n in (Hq + 2 * Hkv, Hq))


@pytest.mark.gpu
@pytest.mark.parametrize("offsets,tokens", WRONG)
def test_nan_throughout(ops, offsets, tokens):
    pk = ops.pack_sequences(torch.tensor(offsets, dtype=torch.int32, device="cuda"), tokens)
    assert ((pk.bounds >= 0) & (pk.bounds <= tokens)).all() and not pk.positions.any()
    for Hq, Hkv, D in HEADS:
        qkv, do = _inputs(tokens, Hq, Hkv, D)
        for causal, window in ((True, 0), (True, 50), (False, 0)):
            out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D, causal, window)
            grad = ops.packed_attn_bwd(do, qkv, torch.zeros_like(do), torch.zeros_like(lse), pk, Hq, Hkv, D, causal, window)
            assert out.isnan().all() and lse.isnan().all() and grad.isnan().all()
    ops.k.check_status()


@pytest.mark.gpu
def test_many_sequences(ops):
    """As many in good order, some of them empty and a tail behind them; two launches instead of one."""
    offsets, tokens = torch.tensor(sorted(MANY + MANY[100:200]), dtype=torch.int32), MANY[-1] + 77
    before = ops.k.launch_count()
    pk, want = ops.pack_sequences(offsets.cuda(), tokens), packed.pack(offsets, tokens)
    assert ops.k.launch_count() - before == 2
    assert torch.equal(pk.bounds.cpu(), want.bounds) and torch.equal(pk.positions.cpu(), want.positions)
    assert (pk.order_tiles[:, 5] == MANY[-1]).all()
    at = torch.tensor(MANY[:packed.PACK_SCAN + 1], dtype=torch.int32)      # the most that one launch does
    before = ops.k.launch_count()
    assert torch.equal(ops.pack_sequences(at.cuda(), tokens).bounds.cpu(), packed.pack(at, tokens).bounds) and ops.k.launch_count() - before == 1
