"""Packed attention with a scale of the caller's own."""
import math

import pytest
import torch

from test_packed_attention import FP32, HALF, _inputs, _offsets, forward64, wrapper  # noqa: F401
from zorse_b200.ops import packed


@pytest.mark.parametrize("scale", [0.0, -0.125, math.inf, math.nan, 1e-40, 1e39])
def test_refused_cpu(wrapper, scale):  # noqa: F811
    T, Hq, Hkv, D = 6, 4, 2, 64
    qkv, do = _inputs(T, Hq, Hkv, D)
    tiles = torch.zeros(1, 8, dtype=torch.int32)
    pk = packed.PackedSequences(T, torch.zeros(256, 2, dtype=torch.int32), torch.zeros(T, dtype=torch.int32), torch.zeros(1, 12, dtype=torch.int32), tiles, tiles)
    with pytest.raises(ValueError, match="scale"):
        wrapper.packed_attn_fwd(qkv, pk, Hq, Hkv, D, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        wrapper.packed_attn_bwd(do, qkv, do, torch.zeros(Hq, T), pk, Hq, Hkv, D, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (64, 16, 64), (2, 2, 128)])
@pytest.mark.parametrize("factor", [0.25, 4.0])
def test_scaled(Hq, Hkv, D, factor):
    """A power of two times the usual scale is the usual attention of queries times that power."""
    from zorse_b200.ops.api import get_ops

    ops, T, lengths = get_ops("sm100"), 700, [300, 0, 350]
    qkv, do = (x.cuda() for x in _inputs(T, Hq, Hkv, D))
    pk = ops.pack_sequences(_offsets(lengths).cuda(), T)
    out, lse = ops.k.packed_attn_fwd(qkv, pk, Hq, Hkv, D, scale=factor / math.sqrt(D))
    times = qkv.clone()
    times[:, :Hq * D] *= factor
    want, lse64, size = forward64(times, lengths, Hq, Hkv, D, True, 0)
    assert ((out.double() - want).abs() <= HALF * (size + want.abs()) + (FP32 + HALF ** 2) * size).all()
    assert ((lse.double() - lse64).abs()[:, :650] <= 4 * FP32).all()      # (scores up to four times as large)
    grad = ops.k.packed_attn_bwd(do, qkv, out, lse, pk, Hq, Hkv, D, scale=factor / math.sqrt(D))
    same = ops.packed_attn_bwd(do, times, out, lse, pk, Hq, Hkv, D)
    assert torch.equal(grad[:, Hq * D:], same[:, Hq * D:])
    assert torch.equal(grad[:, :Hq * D].float(), same[:, :Hq * D].float() * factor)
