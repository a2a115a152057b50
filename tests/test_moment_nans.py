"""Moments in 8 bits: a NaN is held as a NaN, whatever its pattern."""
import pytest
import torch

from zorse_b200.ops import ref
from zorse_b200.ops.api import get_ops
from zorse_b200.ops.moments import Moments8, decode, dither, encode

# quiet NaNs with and without their sign bit, as a CPU's and a GPU's arithmetic make them, and one with every bit set
PATTERNS = [0x7FC00000, -0x400000, 0x7FFFFFFF, -1]


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("add", [0x80000, None])
def test_a_nan_stays_one_cpu(pattern, add):
    nan = torch.tensor([pattern], dtype=torch.int32).view(torch.float32)
    m, v = torch.linspace(-1, 1, 300), torch.linspace(0.5, 1, 300)
    m[7], v[280] = nan, nan
    a, b = decode(encode(m, v, dither(300, 3) if add is None else add))
    assert a[7].isnan() and b[280].isnan()
    assert a.isnan().sum() == 1 and b.isnan().sum() == 1
    held = Moments8.zeros(300)
    held.load(m, v)
    assert decode(held)[0][7].isnan() and decode(held)[1][280].isnan()


def test_a_step_that_makes_a_nan_keeps_it_cpu():
    """An infinite gradient scaled by zero: the NaN of this CPU's arithmetic has its sign bit set."""
    p, g, held = torch.ones(256), torch.ones(256), Moments8.zeros(256)
    g[9] = float("inf")
    kw = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, seed=1)
    ref.adamw_step(p, held, g, step=1, grad_scale=0.0, **kw)
    m, v = decode(held)
    assert p[9].isnan() and m[9].isnan() and v[9].isnan() and not v[10].isnan()
    ref.adamw_step(p, held, torch.ones(256), step=2, **kw)
    assert decode(held)[1][9].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("pattern", PATTERNS)
def test_the_kernel_holds_the_same_codes(pattern):
    nan = torch.tensor([pattern], dtype=torch.int32).view(torch.float32)
    p, g, held = torch.ones(512), torch.linspace(-1, 1, 512), Moments8.zeros(512)
    g[9] = nan
    dev = [p.cuda()], [Moments8(*(t.cuda() for t in held))], [g.cuda()]
    kw = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, seeds=[5])
    get_ops("sm100").adamw_step(*dev, [None], **kw)
    get_ops("ref").adamw_step([p], [held], [g], [None], **kw)
    a, b = (x.cpu() for x in get_ops("sm100").moment_values(dev[1][0]))
    c, d = decode(held)
    assert a[9].isnan() and b[9].isnan() and c[9].isnan() and d[9].isnan()
    rest = torch.arange(512) != 9
    assert torch.equal(a[rest], c[rest]) and torch.equal(b[rest], d[rest])
