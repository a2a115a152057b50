"""Scaled embedding and its gradient by token: sizes that do not fit into 32 bits are refused, and sums over many tokens."""
import pytest
import torch

from zorse_b200.ops import sm100 as k


@pytest.fixture()
def no_launch(monkeypatch):
    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_bf16", lambda t, name: None)
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)


@pytest.mark.parametrize("S,off", [(2 ** 31, 0), (2 ** 32, 0), (2 ** 32 + 6, 2), (6, 2 ** 31), (6, 2 ** 32), (6, 2 ** 31 - 3)])
def test_sequences_and_offsets_beyond_32_bits_are_refused_cpu(no_launch, S, off):
    ids, table, dout = torch.zeros(6, dtype=torch.long), torch.zeros(10, 16, dtype=torch.bfloat16), torch.zeros(6, 16, dtype=torch.bfloat16)
    # (a table of positions as long as asked for, on no device)
    pos = torch.zeros(1, 16, dtype=torch.bfloat16).expand(max(8, min(S, 6) + off), 16)
    pos = type("Rows", (), dict(dtype=pos.dtype, shape=pos.shape, device=pos.device, is_contiguous=lambda self: True,
                                data_ptr=lambda self: 0))()
    with pytest.raises(ValueError, match="2\\^31"):
        k.embedding_scaled(ids, table, pos, S, off, scale=2.0)
    with pytest.raises(ValueError, match="2\\^31"):
        k.embedding_by_token(ids, dout, table, pos, S, off)


def test_the_library_refuses_sizes_it_does_not_count_cpu():
    """Before anything is launched, and before it looks at an address."""
    L = k.lib()
    for H, V, S, off in ((2 ** 31 - 8, 4, 4, 0), (2 ** 30 + 8, 4, 4, 0), (12, 4, 4, 0), (16, -1, 4, 0), (16, 4, -2 ** 31, 0), (16, 4, 4, -1)):
        for call, args in ((L.zb_embedding_scaled, (0, 0, 0, 0, 1, H, V, S, off, 1.0, 0)),
                           (L.zb_embedding_by_token, (0, 0, 0, 0, 0, 1, H, V, S, off, 1.0, 1, 0))):
            assert call(*args) != 0 and L.zb_last_error().startswith(b"embedding: ")


def _shared(call, device):
    buf = torch.zeros(4096, dtype=torch.bfloat16, device=device)
    ids, dout, table = torch.zeros(6, dtype=torch.long, device=device), buf[1024:1120].view(6, 16), torch.zeros(10, 16, dtype=torch.bfloat16, device=device)
    for over in (buf[1024:1184].view(10, 16), buf[1112:1272].view(10, 16), buf[872:1032].view(10, 16), buf[1000:1320].view(torch.float32).view(10, 16)):
        with pytest.raises(ValueError, match="share memory"):
            call(ids, dout, over, None, 6, 0)
    with pytest.raises(ValueError, match="share memory"):
        call(ids, dout, table, buf[1104:1200].view(6, 16), 6, 0)
    return ids, dout, buf[1120:1280].view(10, 16), buf[928:1024].view(6, 16)


def test_a_gradient_in_the_memory_of_its_rows_is_refused_cpu(no_launch):
    args = _shared(k.embedding_by_token, "cpu")
    with pytest.raises(AssertionError, match="was reached"):     # neighbours are not refused
        k.embedding_by_token(*args, 6, 0)


@pytest.mark.gpu
def test_a_gradient_in_the_memory_of_its_rows_is_refused():
    from zorse_b200.ops.api import get_ops

    ops = get_ops("sm100")

    def call(ids, dout, table, pos, S, off):
        ops.embedding_bwd(ids, dout, table, pos, S, off, by_token=True)

    ids, dout, table, pos = _shared(call, "cuda")
    assert ops._embedding_by_token(ids, dout, table, pos, 6, 0, 1.0) is True


@pytest.mark.gpu
def test_without_positions_their_sizes_do_not_matter():
    from zorse_b200.ops.api import get_ops

    ops = get_ops("sm100")
    ids = torch.tensor([3, 1, 3], device="cuda")
    table, dout = torch.randn(5, 16, device="cuda").bfloat16(), torch.ones(3, 16, dtype=torch.bfloat16, device="cuda")
    for S, off in ((0, 0), (2 ** 31, 0), (2 ** 32, -1), (7, 2 ** 40)):
        assert torch.equal(ops.embedding_fwd(ids, table, None, S, off, scale=2.0), (table[ids].float() * 2).bfloat16())
        got = torch.zeros(5, 16, device="cuda")
        ops.embedding_bwd(ids, dout, got, None, S, off, by_token=True)
        assert torch.equal(got.sum(1).cpu(), torch.tensor([0.0, 16, 0, 32, 0]))


def test_the_workspace_of_sizes_it_does_not_count_is_refused_cpu():
    import ctypes

    out = ctypes.c_long(-1)
    for H in (2 ** 31 - 8, 12, 0):
        assert k.lib().zb_embedding_by_token_workspace(4096, H, ctypes.addressof(out)) == -1 and out.value == -1
    assert k.lib().zb_embedding_by_token_workspace(4096, 64, ctypes.addressof(out)) == 0 and out.value > 0
