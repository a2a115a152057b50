"""Head norms backward: a gradient that shares memory with what the pass still reads is refused; rows between rows are not sharing."""
import pytest
import torch

from zorse_b200.ops import sm100 as k


def _view(buf, at, T, W, step):
    return buf.as_strided((T, W), (step, 1), at)


def _addresses(t):
    return {t.data_ptr() + t.element_size() * (r * t.stride(0) + c) for r in range(t.shape[0]) for c in range(t.shape[1])}


def test_which_rows_overlap_cpu():
    """Against sets of addresses; rows of different distances whose stretches meet count as sharing."""
    buf = torch.zeros(400, dtype=torch.bfloat16)
    for T in (1, 2, 3):
        for step in (8, 11, 16):
            a = _view(buf, 100, T, 8, step)
            for at in range(60, 160):
                b = _view(buf, at, T, 8, step)
                want = bool(_addresses(a) & _addresses(b))
                assert k._rows_overlap(a, b) == k._rows_overlap(b, a) == want
    a = _view(buf, 0, 3, 8, 16)
    assert k._rows_overlap(a, _view(buf, 8, 3, 8, 24)) and not k._rows_overlap(a, _view(buf, 40, 3, 8, 24))
    assert not k._rows_overlap(buf[:8], buf[8:16]) and k._rows_overlap(buf[:8], buf[7:15])
    assert not k._rows_overlap(buf[:0], buf[:0])


def _refused(call, T=4, nq=2, nk=1, d=16, device="cpu"):
    W = (nq + 2 * nk) * d
    buf = torch.zeros(4 * T * W + 64, dtype=torch.bfloat16, device=device)
    w, rstd, g = torch.ones(d, dtype=torch.bfloat16, device=device), torch.ones(T, nq + nk, device=device), torch.zeros(4 * d, device=device)
    x = _view(buf, T * W, T, W, W)
    for dy in (x, _view(buf, T * W + W, T, W, W), _view(buf, T * W - 8, T, W, W), _view(buf, T * W + 8, T, W, 2 * W)):
        with pytest.raises(ValueError, match="share memory"):
            call(dy, x, w, w, rstd, None, T, nq, nk, d, g[:d], g[d:2 * d])
    other = torch.zeros(T, W, dtype=torch.bfloat16, device=device)
    for gq, gk in ((g[:d], g[:d]), (g[:d], g[d - 4:2 * d - 4]), (g[8:8 + d], g[:d])):
        with pytest.raises(ValueError, match="share memory"):
            call(other, x, w, w, rstd, None, T, nq, nk, d, gq, gk)


def test_shared_memory_is_refused_cpu(monkeypatch):
    monkeypatch.setattr(k, "_bf16", lambda t, name: None)
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    monkeypatch.setattr(k, "lib", lambda: pytest.fail("the library was reached"))
    _refused(k.qk_norm_rope_bwd)


@pytest.mark.gpu
def test_shared_memory_is_refused_and_rows_between_rows_are_not():
    from zorse_b200.ops.api import get_ops

    ops = get_ops("sm100")
    _refused(ops.qk_norm_rope_bwd, device="cuda")
    T, nq, nk, d = 40, 4, 2, 32
    W = (nq + 2 * nk) * d
    g = torch.Generator().manual_seed(5)
    both = torch.randn(T, 2 * W, generator=g).bfloat16().cuda()
    w = torch.randn(d, generator=g).bfloat16().cuda()
    _, rstd = ops.qk_norm_rope_fwd(both[:, :W], w, w, None, T, nq, nk, d, 1e-5)
    out = []
    for x, dy in ((both[:, :W].clone(), both[:, W:].clone()), (both[:, :W], both[:, W:])):
        gq, gk = torch.zeros(2 * d, device="cuda").chunk(2)
        assert ops._qk_norm_rope_bwd(dy, x, w, w, rstd, None, T, nq, nk, d, gq, gk) is not None
        out.append((dy.clone(), gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(*out))
