"""Attention over packed sequences: what is not a number says so in the row's statistics too."""
import pytest
import torch

from zorse_b200.ops.api import get_ops

T = 700
HEADS = [(4, 1, 64), (4, 2, 64), (2, 2, 64), (6, 3, 64), (8, 1, 128), (2, 2, 128)]


@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_a_nan_in_a_query_is_one_in_its_statistics(ops, Hq, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").bfloat16()
    pk = ops.pack_sequences(torch.tensor([0, 300, 650], dtype=torch.int32, device="cuda"), T)
    want = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
    qkv[310, 3] = float("nan")       # of head 0
    out, lse = ops.packed_attn_fwd(qkv, pk, Hq, Hkv, D)
    assert out[310, :D].isnan().all() and lse[0, 310].isnan()
    here = torch.zeros_like(lse, dtype=torch.bool)
    here[0, 310] = True
    assert torch.equal(lse[~here], want[1][~here]) and torch.equal(out.view(T, Hq, D)[~here.t()], want[0].view(T, Hq, D)[~here.t()])
