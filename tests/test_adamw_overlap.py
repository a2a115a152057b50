"""AdamW over lists: gradients in memory that the step writes.  One in a tensor of its own, element on element, is a matter of order
within a thread; any other would be read after some thread has written there, or not, and is refused."""
import pytest
import torch

from zorse_b200.ops import sm100 as k
from zorse_b200.ops.moments import Moments8

HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)
N = 512


def _lists(bits, dev):
    buf = torch.arange(16 * N, dtype=torch.float32, device=dev) / N
    p = [buf[:N], buf[N:2 * N]]
    moments = [(buf[(2 + 2 * i) * N:(3 + 2 * i) * N], buf[(3 + 2 * i) * N:(4 + 2 * i) * N]) if bits == 32 else Moments8.zeros(N, dev)
               for i in range(2)]
    half = buf[8 * N:10 * N].view(torch.bfloat16)
    return buf, p, moments, [half[:N], half[N:2 * N]]


def _wrong(buf, p, moments, p16, bits):
    """Lists of gradients that overlap what the step writes."""
    good = buf[14 * N:15 * N]
    yield [p[1], good]                                   # another tensor's parameters
    yield [good, buf[4:N + 4]]                           # shifted by a chunk of its own ... of the first tensor
    yield [buf[4:N + 4], good]
    yield [p16[1], good]
    yield [good, p16[0]]
    yield [buf[8 * N:8 * N + N], good]                   # fp32 over both copies in bf16
    yield [buf[:N // 2].view(torch.bfloat16), good]      # bf16 in its own fp32 parameters: not element on element
    if bits == 32:
        yield [moments[1][0], good]
        yield [moments[1][1], moments[0][0]]


def _step(fn, p, moments, g, p16, bits):
    fn(p, moments, g, p16, step=3, seeds=[1, 2] if bits == 8 else None, **HYPER)


def _refusals(fn, bits, dev):
    buf, p, moments, p16 = _lists(bits, dev)
    n = 0
    for g in _wrong(buf, p, moments, p16, bits):
        with pytest.raises(ValueError, match="overlaps"):
            _step(fn, p, moments, g, p16, bits)
        n += 1
    assert n == (9 if bits == 32 else 7)


@pytest.mark.parametrize("bits", [32, 8])
def test_refused_cpu(monkeypatch, bits):
    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    _refusals(k.adamw_step, bits, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_refused_and_a_tensor_of_its_own_is_not(bits):
    from zorse_b200.ops.api import get_ops

    ops = get_ops("sm100")
    _refusals(ops.adamw_step, bits, "cuda")
    for place in ("p", "p16", "m", "v", "same gradient twice"):
        if bits == 8 and place in ("m", "v"):
            continue
        ends = []
        for alias in (False, True):
            buf, p, moments, p16 = _lists(bits, "cuda")
            p16 = [t.copy_(torch.linspace(-1, 1, N)) for t in p16]
            g = {"p": p, "p16": p16, "m": [m[0] for m in moments], "v": [m[-1] for m in moments], "same gradient twice": [buf[14 * N:15 * N]] * 2}[place]
            if not alias:
                g = [t.clone() for t in g]
            native = ops._adamw_step(p, moments, g, p16, [1, 2] if bits == 8 else None, 3, *(HYPER[n] for n in ("lr", "beta1", "beta2", "eps", "weight_decay")), 1.0)
            assert native
            ends.append([t.clone() for t in (*p, *p16, *(x for m in moments for x in m))])
        assert all(torch.equal(a, b) for a, b in zip(*ends))
