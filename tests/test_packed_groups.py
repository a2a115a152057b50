"""The forward kernel for heads of 64 in even groups, at sizes that it is chosen for: four and two heads side by side."""
import math

import pytest
import torch

from test_packed_attention import FP32, HALF, _inputs, _offsets, forward64
from zorse_b200.ops.api import get_ops

CASES = [  # T, lengths, query heads, key heads, causal, window
    (640, [100, 90, 0, 260], 64, 16, True, 0), (513, [1] * 300 + [0, 65, 64, 63], 128, 8, True, 0), (700, [64, 64, 500, 60], 64, 8, True, 65),
    (1000, [999], 60, 15, True, 1), (600, [129, 60, 127, 200], 80, 20, False, 0), (129, [], 160, 2, False, 0), (1100, [1000, 77], 32, 4, True, 150),
    (3000, [1290, 5, 1705], 16, 4, True, 0),
    (640, [100, 90, 0, 260], 160, 80, True, 0), (1031, [130, 700, 191], 102, 17, True, 0), (900, [1] * 200 + [64, 0, 65, 500], 130, 13, True, 37),
    (513, [510], 170, 85, False, 0), (1300, [1300], 90, 45, True, 400), (5000, [2500, 100, 2390], 30, 3, True, 0),
]


@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_forward(ops, case):
    T, lengths, Hq, Hkv, causal, window = case
    # more than a round of CTAs of 256 rows (three where two heads are side by side), on the GPU that this is for
    assert Hq // Hkv % 2 == 0 and Hq * -(-T // 256) > (148 if Hq // Hkv % 4 == 0 else 3 * 148)
    qkv, _ = (x.cuda() for x in _inputs(T, Hq, Hkv, 64))
    total = sum(lengths)
    qkv[total:] = float("nan")
    pk = ops.pack_sequences(_offsets(lengths).cuda(), T)
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, 64, causal, window)
    want, lse64, size = forward64(qkv, lengths, Hq, Hkv, 64, causal, window)
    assert ((out.double() - want).abs() <= HALF * (size + want.abs()) + (FP32 + HALF ** 2) * size).all()
    assert torch.equal(lse.isinf(), lse64.isinf()) and ((lse.double() - lse64).abs()[:, :total] <= FP32).all()
    assert (out[total:] == 0).all()
    again = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, 64, causal, window)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    ops.k.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(64, 16), (160, 80)])
def test_nan(ops, Hq, Hkv):
    """Offsets that do not rise: throughout.  In a query: its own row."""
    T = 700
    qkv, _ = (x.cuda() for x in _inputs(T, Hq, Hkv, 64))
    out, lse = ops.packed_attn_fwd(qkv, ops.pack_sequences(torch.tensor([0, 300, 200, T], dtype=torch.int32, device="cuda"), T), Hq, Hkv, 64)
    assert out.isnan().all() and lse.isnan().all()
    pk = ops.pack_sequences(_offsets([300, 350]).cuda(), T)
    want = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, 64)
    qkv[310, 3] = float("nan")
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, 64)
    assert out[310, :64].isnan().all() and lse[0, 310].isnan() and lse.isnan().sum() == 1 and out.isnan().sum() == 64
    there = ~lse.isnan()
    assert torch.equal(lse[there], want[1][there]) and math.isinf(lse[0, 690])


@pytest.mark.gpu
def test_both_kernels_by_size(ops):
    """The same sequences under few tokens (two chains a CTA) and many (four): as near to each other as either is to the exact result."""
    Hq, Hkv, n = 8, 2, 256
    qkv, _ = (x.cuda() for x in _inputs(40 * n, Hq, Hkv, 64))
    few, lse = ops.packed_attn_fwd(qkv[:n], ops.pack_sequences(_offsets([n]).cuda(), n), Hq, Hkv, 64)
    many, lse2 = ops.packed_attn_fwd(qkv, ops.pack_sequences(_offsets([n] * 40).cuda(), 40 * n), Hq, Hkv, 64)
    _, _, size = forward64(qkv[:n], [n], Hq, Hkv, 64, True, 0)
    assert ((few.double() - many[:n].double()).abs() <= 2 * (2 * HALF + FP32 + HALF ** 2) * size).all()
    assert ((lse - lse2[:, :n]).abs() <= 2 * FP32).all()
