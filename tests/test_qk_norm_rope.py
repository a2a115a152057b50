"""Head norms with the rotation in the same pass: against the formulas in 64 bits, against differences, and what is refused."""
import pytest
import torch

from zorse_b200.ops import ref
from zorse_b200.ops.api import get_ops

HALF = 2.0 ** -8          # half a step of bf16, relative


def _inputs(T, nq, nk, d, S, rope=True, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0, at=0.0):
        return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + at).to(dtype)

    cs = ref.rope_table(S, d, 10000.0) if rope else None
    return normal(T, (nq + 2 * nk) * d), normal(d, scale=0.3, at=1.0), normal(d, scale=0.3, at=1.0), cs, normal(T, (nq + 2 * nk) * d)


def _turn64(x, cs, S, sign):
    if cs is None:
        return x
    h = x.shape[-1] // 2
    at = torch.arange(x.shape[0]) % S
    c, s = cs.double()[at, None, :h], cs.double()[at, None, h:] * sign
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def _fwd64(qkv, wq, wk, cs, S, nq, nk, d, eps):
    """(rotated heads, 1 / rms, normalised heads)"""
    x = qkv.double()[:, :(nq + nk) * d].view(-1, nq + nk, d)
    w = torch.cat([wq.double().expand(nq, d), wk.double().expand(nk, d)])
    r = (x.square().mean(-1) + eps) ** -0.5
    n = x * r[..., None] * w
    return _turn64(n, cs, S, 1.0), r, n


SHAPES = [  # T, q heads, kv heads, width, S
    (1, 1, 1, 64, 1), (3, 2, 1, 128, 3), (130, 8, 8, 64, 65), (257, 5, 3, 96, 257), (64, 4, 2, 256, 16), (19, 3, 1, 16, 7),
    (33, 2, 2, 512, 33), (40, 7, 1, 48, 50), (2000, 32, 8, 128, 1000),
    (50, 3, 0, 64, 50), (50, 0, 2, 128, 25), (37, 4, 1, 64, 3), (1001, 2, 2, 128, 333), (5, 1, 1, 32, 9), (613, 8, 4, 64, 613), (4099, 1, 1, 16, 2),
]


@pytest.mark.parametrize("rope", [True, False])
def test_formulas_and_differences_cpu(rope):
    """The reference backend in 64-bit inputs: forward by the formula, gradients by differences."""
    T, nq, nk, d, S, eps = 5, 3, 2, 16, 4, 1e-5
    qkv, wq, wk, cs, dy = _inputs(T, nq, nk, d, S, rope, dtype=torch.float32)
    ops = get_ops("ref")
    out, rstd = ops.qk_norm_rope_fwd(qkv, wq, wk, cs, S, nq, nk, d, eps)
    want, r, _ = _fwd64(qkv, wq, wk, cs, S, nq, nk, d, eps)
    cut = (nq + nk) * d
    assert torch.allclose(out[:, :cut].double(), want.reshape(T, cut), atol=1e-5)
    assert torch.equal(out[:, cut:], qkv[:, cut:]) and torch.allclose(rstd.double(), r, rtol=1e-5)
    gq, gk = torch.zeros(d), torch.zeros(d)
    dx = ops.qk_norm_rope_bwd(dy.clone(), qkv, wq, wk, rstd, cs, S, nq, nk, d, gq, gk)
    assert torch.equal(dx[:, cut:], dy[:, cut:])

    def loss(q, a, b):
        return float((_fwd64(q, a, b, cs, S, nq, nk, d, eps)[0].reshape(T, cut) * dy[:, :cut].double()).sum())

    h = 1e-4
    for i, j in [(0, 0), (4, 9), (2, cut - 1), (3, 17), (1, 30), (4, nq * d + 3)]:
        step = torch.zeros_like(qkv, dtype=torch.float64)
        step[i, j] = h
        diff = (loss(qkv.double() + step, wq, wk) - loss(qkv.double() - step, wq, wk)) / (2 * h)
        assert abs(diff - float(dx[i, j])) < 1e-4 * (1 + abs(diff))
    for j in (0, 5, d - 1):
        step = torch.zeros(d, dtype=torch.float64)
        step[j] = h
        dq = (loss(qkv, wq.double() + step, wk) - loss(qkv, wq.double() - step, wk)) / (2 * h)
        dk = (loss(qkv, wq, wk.double() + step) - loss(qkv, wq, wk.double() - step)) / (2 * h)
        assert abs(dq - float(gq[j])) < 1e-4 * (1 + abs(dq)) and abs(dk - float(gk[j])) < 1e-4 * (1 + abs(dk))


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
    T, nq, nk, d, S = 6, 2, 1, 64, 3
    qkv, wq, wk, cs, dy = _inputs(T, nq, nk, d, S)
    ok = dict(qkv=qkv, wq=wq, wk=wk, cs=cs, S=S, nq=nq, nk=nk, d=d, eps=1e-5)
    for wrong in (dict(qkv=qkv[:, :-8]), dict(qkv=qkv.t().contiguous().t()), dict(wq=wq[:32]), dict(wk=wk.repeat(2)[::2]),
                  dict(cs=cs.double()), dict(cs=cs[:2]), dict(cs=cs[:, :32].contiguous()), dict(qkv=qkv.view(-1)), dict(S=0)):
        with pytest.raises(ValueError):
            wrapper.qk_norm_rope_fwd(**{**ok, **wrong})
    with pytest.raises(TypeError):
        wrapper.qk_norm_rope_fwd(**{**ok, "wq": wq.float()})
    ok.pop("eps")
    g, rstd = torch.zeros(d), torch.ones(T, nq + nk)
    ok |= dict(dqkv=dy, rstd=rstd, gwq=g, gwk=g.clone())
    for wrong in (dict(dqkv=qkv), dict(dqkv=dy[:3]), dict(rstd=rstd[:, :2]), dict(rstd=rstd.double()), dict(gwq=g.bfloat16()),
                  dict(gwq=g.double(), gwk=g.double()), dict(gwk=g[:32]), dict(gwk=g)):
        with pytest.raises(ValueError):
            wrapper.qk_norm_rope_bwd(**{**ok, **wrong})


# ---------------------------------------------------------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


# A head's sum of squares is added in chains of 16 and then over lanes: at most 2^-19 relative with the reciprocal root's 2^-22,
# products and the rotation add a few 2^-24 of the values that they combine.
FP32 = 2.0 ** -18


@pytest.mark.gpu
@pytest.mark.parametrize("T,nq,nk,d,S", SHAPES)
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("keep", [True, False])
def test_forward(ops, T, nq, nk, d, S, rope, keep):
    qkv, wq, wk, cs, _ = _inputs(T, nq, nk, d, S, rope)
    a, b, c, t = _cuda(qkv, wq, wk, cs)
    out, rstd = ops.qk_norm_rope_fwd(a, b, c, t, S, nq, nk, d, 1e-5, keep=keep)
    want, r, n = _fwd64(qkv, wq, wk, cs, S, nq, nk, d, 1e-5)
    cut = (nq + nk) * d
    assert torch.equal(out[:, cut:].cpu(), qkv[:, cut:])
    got = out[:, :cut].cpu().double().view(T, nq + nk, d)
    size = n.abs() + n.abs().roll(d // 2, -1)
    assert ((got - want).abs() <= HALF * want.abs() + FP32 * size).all()
    if keep:
        assert torch.equal(a.cpu(), qkv)
        assert ((rstd.cpu().double() - r).abs() <= FP32 * r).all()
    else:
        assert out.data_ptr() == a.data_ptr() and rstd is None


def _bwd64(qkv, wq, wk, cs, dy, S, nq, nk, d, eps):
    """dx, dwq, dwk, and for each the size of what is added up."""
    T = qkv.shape[0]
    cut = (nq + nk) * d
    x = qkv.double()[:, :cut].view(T, nq + nk, d)
    w = torch.cat([wq.double().expand(nq, d), wk.double().expand(nk, d)])
    r = (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    g0 = dy.double()[:, :cut].view(T, nq + nk, d)
    g = _turn64(g0, cs, S, -1.0)
    ga = g0.abs() + g0.abs().roll(d // 2, -1)
    xh = x * r
    dx = r * (w * g - xh * (w * g * xh).mean(-1, keepdim=True))
    dxa = r * (w.abs() * ga + xh.abs() * (w.abs() * ga * xh.abs()).mean(-1, keepdim=True))
    dw, dwa = (g * xh).sum(0), (ga * xh.abs()).sum(0)
    return dx, dxa, dw[:nq].sum(0), dwa[:nq].sum(0), dw[nq:].sum(0), dwa[nq:].sum(0), r[..., 0]


@pytest.mark.gpu
@pytest.mark.parametrize("T,nq,nk,d,S", SHAPES)
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
def test_backward(ops, T, nq, nk, d, S, rope, grads):
    qkv, wq, wk, cs, dy = _inputs(T, nq, nk, d, S, rope)
    dx, dxa, dq, dqa, dk, dka, r = _bwd64(qkv, wq, wk, cs, dy, S, nq, nk, d, 1e-5)
    sq, sk = torch.linspace(-1, 1, d).to(grads), torch.linspace(2, 1, d).to(grads)
    a, b, c, t, g, gq, gk = _cuda(qkv, wq, wk, cs, dy, sq, sk)
    got = ops.qk_norm_rope_bwd(g, a, b, c, r.float().cuda(), t, S, nq, nk, d, gq, gk)
    cut = (nq + nk) * d
    assert got.data_ptr() == g.data_ptr() and torch.equal(got[:, cut:].cpu(), dy[:, cut:]) and torch.equal(a.cpu(), qkv)
    diff = (got[:, :cut].cpu().double().view(T, nq + nk, d) - dx).abs()
    assert (diff <= HALF * dx.abs() + FP32 * dxa).all()
    half = torch.finfo(grads).eps / 2
    for got, slot, want, size in ((gq, sq, dq, dqa), (gk, sk, dk, dka)):
        want = slot.double() + want
        # the longest chain of fp32 additions here is far below 256
        assert ((got.cpu().double() - want).abs() <= half * want.abs() + (FP32 + 256 * 2.0 ** -24) * size + 2.0 ** -23 * slot.double().abs()).all()


@pytest.mark.gpu
def test_strided_rows_streams_and_repeats(ops):
    """Rows inside a wider buffer whose other columns stay; another stream; the same bits twice; a captured graph."""
    T, nq, nk, d, S = 70, 4, 2, 128, 70
    qkv, wq, wk, cs, dy = _inputs(T, nq, nk, d, S)
    width = (nq + 2 * nk) * d
    wide = torch.full((T, width + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 32:32 + width] = qkv.cuda()
    b, c, t = _cuda(wq, wk, cs)
    want, rstd = ops.qk_norm_rope_fwd(qkv.cuda(), b, c, t, S, nq, nk, d, 1e-5)
    out, r2 = ops.qk_norm_rope_fwd(wide[:, 32:32 + width], b, c, t, S, nq, nk, d, 1e-5)
    assert torch.equal(out, want) and torch.equal(r2, rstd)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.qk_norm_rope_fwd(wide[:, 32:32 + width], b, c, t, S, nq, nk, d, 1e-5, keep=False)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(wide[:, 32:32 + width], want) and (wide[:, :32] == 7).all() and (wide[:, 32 + width:] == 7).all()

    def backward():
        g, gq, gk = dy.cuda(), torch.ones(d, device="cuda"), torch.ones(d, device="cuda")
        ops.qk_norm_rope_bwd(g, qkv.cuda(), b, c, rstd, t, S, nq, nk, d, gq, gk)
        return g, gq, gk

    first = backward()
    assert all(torch.equal(x, y) for x, y in zip(first, backward()))
    a, src, g, gq, gk = qkv.cuda(), dy.cuda(), torch.empty_like(dy, device="cuda"), torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g.copy_(src)
        gq.fill_(1.0)
        gk.fill_(1.0)
        ops.qk_norm_rope_bwd(g, a, b, c, rstd, t, S, nq, nk, d, gq, gk)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(first, (g, gq, gk)))


@pytest.mark.gpu
def test_edges(ops):
    """No tokens; a head of zeros; NaN and infinity stay in their head."""
    d = 64
    qkv, wq, wk, cs, _ = _inputs(4, 2, 1, d, 4)
    b, c, t = _cuda(wq, wk, cs)
    out, rstd = ops.qk_norm_rope_fwd(qkv[:0].cuda(), b, c, t, 4, 2, 1, d, 1e-5)
    assert out.shape == (0, 4 * d) and rstd.shape == (0, 3)
    gq = torch.ones(d, device="cuda")
    ops.qk_norm_rope_bwd(out.clone(), out, b, c, rstd, t, 4, 2, 1, d, gq, gq.clone())
    assert (gq == 1).all()
    qkv[0, :d] = 0
    qkv[1, d] = float("nan")
    qkv[2, 0] = float("inf")
    out, rstd = ops.qk_norm_rope_fwd(qkv.cuda(), b, c, t, 4, 2, 1, d, 1e-5)
    heads = out.float().cpu().view(4, 4, d)
    assert (heads[0, 0] == 0).all() and heads[1, 1].isnan().all() and not heads[2, 0].isfinite().all()
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[1, 1] = bad[2, 0] = True
    assert heads[~bad].isfinite().all()


@pytest.mark.gpu
def test_refused_by_the_library(ops):
    from zorse_b200.ops.sm100 import KernelError

    x = torch.zeros(4, 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(72, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError):        # a head width that is no multiple of 16
        ops.qk_norm_rope_fwd(torch.zeros(4, 4 * 72, dtype=torch.bfloat16, device="cuda"), w, w, None, 4, 2, 1, 72, 1e-5)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError):        # rows to write that lie over one another
        ops.qk_norm_rope_fwd(x[:1, :256].expand(4, 256), w[:64], w[:64], None, 4, 2, 1, 64, 1e-5, keep=False)
    with pytest.raises(KernelError):        # rows off a 16-byte boundary
        ops.qk_norm_rope_fwd(x[:, 1:1 + 256], w, w, None, 4, 2, 1, 64, 1e-5)
    with pytest.raises(KernelError):        # a row stride that is no multiple of 8
        ops.qk_norm_rope_fwd(torch.zeros(4, 260, dtype=torch.bfloat16, device="cuda")[:, :256], w, w, None, 4, 2, 1, 64, 1e-5)
