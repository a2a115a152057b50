"""AdamW over lists of tensors with moments in 32 bits or 8: against 64 bits, bit for bit against the reference backend, what the
codes can hold, and what is refused."""
import math

import pytest
import torch

from zorse_b200.ops.api import get_ops
from zorse_b200.ops.moments import BLOCK, Moments8, decode, dither, dither_seed, encode

HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, grad_scale=0.5)


def _tensors(sizes, bits, gdt, seed=0, fresh=False):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=g) for n in sizes]
    grads = [(torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g)) * 1e-2).to(gdt) for n in sizes]
    moments = []
    for n in sizes:
        m, v = torch.randn(n, generator=g) * 1e-2, torch.randn(n, generator=g).square() * 1e-4
        if fresh:
            m, v = torch.zeros(n), torch.zeros(n)
        moments.append((m, v) if bits == 32 else encode(m, v))
    p16 = [torch.full((n,), 5.0, dtype=torch.bfloat16) for n in sizes]
    return p, moments, grads, p16


def _step64(p, mv, g, *, lr, beta1, beta2, eps, weight_decay, grad_scale, step):
    """(p, m, v) in 64 bits, and the size of the update."""
    m, v = (t.double() for t in mv)
    g = g.double() * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    up = lr / (1 - beta1 ** step) * m / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return p.double() * (1 - lr * weight_decay) - up, m, v, up.abs()


# ------------------------------------------------------------------------------------------------------------------- codes
def test_codes_are_exact_and_stable_cpu():
    g = torch.Generator().manual_seed(1)
    for n in (1, 255, 256, 257, 5000):
        m = torch.randn(n, generator=g) * torch.exp(3 * torch.randn(n, generator=g))
        v = (torch.randn(n, generator=g) * torch.exp(3 * torch.randn(n, generator=g))).square() * 1e-9
        c = encode(m, v)
        a, b = decode(c)
        assert torch.equal(a.bfloat16().float(), a) and torch.equal(b.bfloat16().float(), b)
        blocks = torch.nn.functional.pad(m.abs(), (0, -n % BLOCK)).view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)[:n]
        near = m.abs() > blocks * 2.0 ** -14               # those further below the block's largest may become zero
        assert ((a - m).abs()[near] <= 2.0 ** -4 * m.abs()[near]).all() and (a.abs()[~near] <= m.abs()[~near] * (1 + 2.0 ** -4)).all()
        # 255 codes, eight to a binade: code 1 lies 31.75 binades below the block's largest, or up to one code less (the base is
        # rounded up); what is smaller is held as code 1
        top = torch.nn.functional.pad(v, (0, -n % BLOCK)).view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)[:n]
        far = v < top * 2.0 ** -31
        assert ((b - v).abs()[~far] <= 2.0 ** -4 * v[~far]).all() and (b[far] <= top[far] * 2.0 ** -30).all() and (b[v > 0] > 0).all()
        again = decode(encode(a, b))
        assert torch.equal(again[0], a) and torch.equal(again[1], b)
    z = Moments8.zeros(300)
    assert all((t == 0).all() for t in decode(z)) and z.m_base.numel() == 2
    z.load(torch.full((300,), -2.0), torch.full((300,), 3.0))
    assert (decode(z)[0] == -2).all() and (decode(z)[1] == 3).all()


def test_special_values_cpu():
    x = torch.tensor([float("inf"), float("nan"), -float("inf"), 0.0])
    m, v = decode(encode(x, torch.tensor([float("inf"), float("nan"), 0.0, 1.0])))
    assert m[0] == math.inf and m[1].isnan() and m[2] == -math.inf and m[3] == 0 and v[0] == math.inf and v[1].isnan() and v[2] == 0


def test_dither_is_even_cpu():
    """The expectation of what is held is the value: 2^14 seeds, a standard error of a code's width / sqrt(12 * 2^14) at most."""
    x = torch.tensor([1.03, 1.0001, 3.7, 0.9])
    held = torch.stack([decode(encode(x, x, dither(4, dither_seed(s, 5), None)))[0] for s in range(1 << 12)]).double()
    width = 2.0 ** (torch.floor(torch.log2(x.double())) - 3)
    assert ((held.mean(0) - x.double()).abs() <= 6 * 0.5 * width / math.sqrt(1 << 12) + 2.0 ** -16 * width).all()
    d = dither(100001, 7)
    assert d.numel() == 100001 and int(d.min()) >= 8 and int(d.max()) <= 0xFFFF8 and (d & 15 == 8).all()
    assert abs(float(d.double().mean()) / 0x80000 - 1) < 6 / math.sqrt(3 * 100001)


def test_moments_reach_a_constant_gradient_cpu():
    """Rounded to nearest, v would stand still far below the gradient's square; dithered, its mean is the unrounded moment."""
    n, ops = 4096, get_ops("ref")
    p, g, mom = [torch.zeros(n)], [torch.full((n,), 0.37)], [Moments8.zeros(n)]
    steps, b2 = 400, 0.99
    for k in range(1, steps + 1):
        ops.adamw_step(p, mom, g, [None], lr=1e-3, beta1=0.9, beta2=b2, eps=1e-8, weight_decay=0.0, step=k, seeds=[dither_seed(k)])
    m, v = (t.double() for t in ops.moment_values(mom[0]))
    want = 0.37 ** 2 * (1 - b2 ** steps)
    # each step adds a rounding of variance at most (an eighth)^2 / 4 relative, damped by b2^2 a step: 0.44 relative, over 64
    assert abs(float(v.mean()) / want - 1) < 6 * 0.44 / 64
    assert abs(float(m.mean()) / 0.37 - 1) < 6 * 0.15 / 64


def test_reference_backend_cpu():
    sizes = [1, 300, 1000]
    for bits in (32, 8):
        p, moments, g, p16 = _tensors(sizes, bits, torch.float32)
        before = [(x.clone(), decode(m) if bits == 8 else tuple(t.clone() for t in m)) for x, m in zip(p, moments)]
        get_ops("ref").adamw_step(p, moments, g, p16, step=[3, 1, 7], seeds=[1, 2, 3] if bits == 8 else None, **HYPER)
        for i, (x, mv) in enumerate(before):
            want, m, v, up = _step64(x, mv, g[i], step=[3, 1, 7][i], **HYPER)
            assert ((p[i].double() - want).abs() <= 2.0 ** -22 * (want.abs() + up) + 2.0 ** -23 * x.double().abs()).all()
            assert torch.equal(p16[i], p[i].bfloat16())
            if bits == 32:
                assert torch.allclose(moments[i][0].double(), m, rtol=1e-5, atol=1e-9) and torch.allclose(moments[i][1].double(), v, rtol=1e-5)


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refusals_cpu(monkeypatch):
    from zorse_b200.ops import sm100 as k

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)

    def call(bits=32, **wrong):
        p, moments, g, p16 = _tensors([300, 40], bits, torch.float32)
        a = dict(p=p, moments=moments, g=g, p16=p16, step=1, seeds=[1, 2], **HYPER)
        a.update({name: f(a[name]) for name, f in wrong.items()})
        k.adamw_step(a.pop("p"), a.pop("moments"), a.pop("g"), a.pop("p16"), **a)

    def swap(i, x):
        return lambda old: [x if j == i else t for j, t in enumerate(old)]

    for wrong in (dict(p=lambda p: p[:1]), dict(g=lambda g: g[:1]), dict(p16=lambda c: c[:1]), dict(step=lambda s: 0),
                  dict(step=lambda s: [1]), dict(step=lambda s: [3, 0]), dict(p=swap(0, torch.zeros(300).double())),
                  dict(p=lambda p: [p[0], p[0][:40]]), dict(p=swap(0, torch.zeros(600)[::2])), dict(g=swap(1, torch.zeros(39))),
                  dict(g=swap(1, torch.zeros(40).half())), dict(p16=swap(0, torch.zeros(300))), dict(p16=swap(0, torch.zeros(299).bfloat16())),
                  dict(beta1=lambda b: 1.0), dict(beta2=lambda b: -0.1), dict(p=lambda p: [p[0], p[0][100:140]]),
                  dict(moments=lambda m: [m[0], (m[0][0][:40], torch.zeros(40))]),
                  dict(moments=swap(1, (torch.zeros(40), torch.zeros(41)))), dict(moments=swap(1, (torch.zeros(40).bfloat16(), torch.zeros(40))))):
        with pytest.raises(ValueError):
            call(**wrong)
    for wrong in (dict(seeds=lambda s: None), dict(seeds=lambda s: [1]), dict(moments=swap(0, Moments8.zeros(299))),
                  dict(moments=swap(0, Moments8.zeros(300)._replace(m_base=torch.zeros(1, dtype=torch.int16)))),
                  dict(moments=swap(0, Moments8.zeros(300)._replace(v=torch.zeros(300))))):
        with pytest.raises(ValueError):
            call(8, **wrong)
    p, moments, g, p16 = _tensors([300, 40], 8, torch.float32)
    with pytest.raises(ValueError):          # moments of both kinds in one list
        k.adamw_step(p, [moments[0], (torch.zeros(40), torch.zeros(40))], g, p16, step=1, seeds=[1, 2], **HYPER)
    k.adamw_step([], [], [], [], step=1, **HYPER)
    for bad in (dict(v=torch.zeros(299, dtype=torch.uint8)), dict(v_base=torch.zeros(2)), dict(m_base=torch.zeros(3, dtype=torch.int16))):
        with pytest.raises(ValueError):
            k.moment_values(Moments8.zeros(300)._replace(**bad))
    with pytest.raises(ValueError):
        k.moment_values(Moments8.zeros(300), torch.float16)


# ---------------------------------------------------------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def ops():
    return get_ops("sm100")


def _to(x, dev):
    if isinstance(x, Moments8):
        return Moments8(*(t.to(dev) for t in x))
    if isinstance(x, (list, tuple)):
        return type(x)(_to(t, dev) for t in x)
    return None if x is None else x.to(dev)


LISTS = [[1], [4], [5, 3], [256], [257, 255], [2048, 2049, 7], [300000], [1000 + 13 * i for i in range(40)], [640 + i for i in range(300)]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fresh", [True, False])
def test_step(ops, sizes, bits, gdt, fresh):
    """Moments bit for bit those of the reference backend, whose operations round one by one as well; parameters within the
    errors of the fast quotient and root (2^-22 each) of the update."""
    p, moments, g, p16 = _tensors(sizes, bits, gdt, fresh=fresh)
    p16[-1] = None
    steps = [1 + 5 * i for i in range(len(sizes))]
    seeds = [dither_seed(7, i) for i in range(len(sizes))] if bits == 8 else None
    dev = [_to(x, "cuda") for x in (p, moments, g, p16)]
    old = [(x.clone(), decode(m) if bits == 8 else tuple(t.clone() for t in m)) for x, m in zip(p, moments)]
    ops.adamw_step(*dev, step=steps, seeds=seeds, **HYPER)
    get_ops("ref").adamw_step(p, moments, g, p16, step=steps, seeds=seeds, **HYPER)
    for i in range(len(sizes)):
        for a, b in zip(dev[1][i], moments[i]):
            assert torch.equal(a.cpu(), b)
        want, _, _, up = _step64(old[i][0], old[i][1], g[i], step=steps[i], **HYPER)
        got = dev[0][i].cpu()
        assert ((got.double() - want).abs() <= 2.0 ** -23 * (old[i][0].double().abs() + want.abs()) + 2.0 ** -19 * up).all()
        if p16[i] is not None:
            assert torch.equal(dev[3][i].cpu(), got.bfloat16())
        assert torch.equal(dev[2][i].cpu(), g[i])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_in_a_row_and_neighbours(ops, bits):
    """Twenty steps on slices of one buffer: the moments stay those of the reference backend, and nothing between the slices moves."""
    sizes, starts = [1000, 70, 513], [0, 1024, 1280]
    p, moments, g, p16 = _tensors(sizes, bits, torch.float32, fresh=True)
    buf = torch.full((2048,), 3.0, device="cuda")
    dev_p = [buf[o:o + n].copy_(x) for o, n, x in zip(starts, sizes, p)]
    dev_m = _to(moments, "cuda")
    for k in range(1, 21):
        gk = [x * math.cos(k) for x in g]
        seeds = [dither_seed(k, i) for i in range(3)] if bits == 8 else None
        ops.adamw_step(dev_p, dev_m, _to(gk, "cuda"), [None] * 3, step=k, seeds=seeds, **HYPER)
        get_ops("ref").adamw_step(p, moments, gk, [None] * 3, step=k, seeds=seeds, **HYPER)
    for a, b in zip(dev_m, moments):
        assert all(torch.equal(x.cpu(), y) for x, y in zip(a, b))
    used = torch.zeros(2048, dtype=torch.bool, device="cuda")
    for o, n in zip(starts, sizes):
        used[o:o + n] = True
    assert (buf[~used] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_both_types_in_one_list_and_empty_tensors(ops, bits):
    sizes = [700, 0, 5000, 256, 33]
    p, moments, g, p16 = _tensors(sizes, bits, torch.float32)
    g = [x.bfloat16() if i % 2 else x for i, x in enumerate(g)]
    g[2] = g[2].bfloat16()
    seeds = [3, 4, 5, 6, 7] if bits == 8 else None
    dev = [_to(x, "cuda") for x in (p, moments, g, p16)]
    ops.adamw_step(*dev, step=2, seeds=seeds, **HYPER)
    get_ops("ref").adamw_step(p, moments, g, p16, step=2, seeds=seeds, **HYPER)
    for a, b in zip(dev[1], moments):
        assert all(torch.equal(x.cpu(), y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_that_follow_at_once_on_other_processors(ops, bits):
    """Launches that begin under the end of the one before: blocks that share lines of bases, and whole tensors, go to other
    processors from step to step (the list turned round), with nothing in between."""
    sizes = [400000, 90000, 257, 130000]
    p, moments, g, p16 = _tensors(sizes, bits, torch.float32, fresh=True)
    dev = [_to(x, "cuda") for x in (p, moments, g, p16)]
    steps = [(k, [dither_seed(k, i) for i in range(4)] if bits == 8 else None) for k in range(1, 9)]
    for k, seeds in steps:
        turn = slice(None, None, -1 if k % 2 else 1)
        ops.adamw_step(*(x[turn] for x in dev), step=k, seeds=seeds and seeds[turn], **HYPER)
    for k, seeds in steps:
        get_ops("ref").adamw_step(p, moments, g, p16, step=k, seeds=seeds, **HYPER)
    for a, b in zip(dev[1], moments):
        assert all(torch.equal(x.cpu(), y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_special_gradients(ops):
    """Infinities and NaN show in the moments that they reach and in no other block."""
    n = 3 * BLOCK
    p, moments, g, p16 = _tensors([n], 8, torch.float32, fresh=True)
    g[0][5], g[0][300] = float("inf"), float("nan")
    dev = [_to(x, "cuda") for x in (p, moments, g, p16)]
    ops.adamw_step(*dev, step=1, seeds=[9], **HYPER)
    get_ops("ref").adamw_step(p, moments, g, p16, step=1, seeds=[9], **HYPER)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev[1][0], moments[0]))
    m, v = (t.cpu() for t in ops.moment_values(dev[1][0]))
    assert m[5] == math.inf and v[5] == math.inf and m[300].isnan() and v[300].isnan()
    assert m[2 * BLOCK:].isfinite().all() and (v[2 * BLOCK:] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 256, 1027, 100000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_moment_values(ops, n, dtype):
    code = encode(torch.randn(n, generator=torch.Generator().manual_seed(1)), torch.rand(n, generator=torch.Generator().manual_seed(2)))
    for a, b in zip(ops.moment_values(_to(code, "cuda"), dtype), decode(code)):
        assert a.dtype == dtype and torch.equal(a.float().cpu(), b)


@pytest.mark.gpu
def test_captured_graph_and_other_stream(ops):
    sizes = [5000, 33]
    p, moments, g, p16 = _tensors(sizes, 8, torch.bfloat16)
    a, b = ([_to(x, "cuda") for x in (p, moments, g, p16)] for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            ops.adamw_step(*a, step=4, seeds=[1, 2], **HYPER)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.adamw_step(*b, step=4, seeds=[1, 2], **HYPER)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(a[1] + [a[0], a[3]], b[1] + [b[0], b[3]]):
        assert all(torch.equal(t, u) for t, u in zip(x, y))


@pytest.mark.gpu
def test_refused_by_the_library(ops):
    from zorse_b200.ops.sm100 import KernelError

    p, moments, g, p16 = (_to(x, "cuda") for x in _tensors([256], 32, torch.float32))
    off = torch.zeros(257, device="cuda")[1:]
    with pytest.raises(KernelError):
        ops.adamw_step([off], moments, g, p16, step=1, **HYPER)
    with pytest.raises(KernelError):
        ops.adamw_step(p, [(off, off.clone())], g, p16, step=1, **HYPER)
