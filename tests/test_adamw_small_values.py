"""AdamW over lists where second moments are subnormal: the root must not take them as zero."""
import math

import pytest
import torch

from zorse_b200.ops.api import get_ops
from zorse_b200.ops.moments import Moments8, decode, dither_seed

HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.999, weight_decay=0.1)
SIZES = [700, 256, 33]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-24])
@pytest.mark.parametrize("size", [1e-18, 3e-20])
def test_second_moments_below_the_normal_numbers(bits, eps, size):
    """Gradients of 1e-18 give v of 1e-39, a subnormal number.  The moments keep the reference backend's bits; the update is
    computed in 64 bits from m and v rounded as the step rounds them."""
    dev, ref = get_ops("sm100"), get_ops("ref")
    g = torch.Generator().manual_seed(11)
    p = [torch.randn(n, generator=g) * 1e-3 for n in SIZES]
    moments = [Moments8.zeros(n) if bits == 8 else (torch.zeros(n), torch.zeros(n)) for n in SIZES]
    on_gpu = [x.cuda() for x in p], [type(m)(*(t.cuda() for t in m)) if bits == 8 else tuple(t.cuda() for t in m) for m in moments]
    b1, b2, lr = HYPER["beta1"], HYPER["beta2"], HYPER["lr"]
    for k in range(1, 4):
        grads = [size * (1 + torch.rand(n, generator=g)) * (torch.rand(n, generator=g) - 0.5).sign() for n in SIZES]
        seeds = [dither_seed(k, i) for i in range(len(SIZES))] if bits == 8 else None
        old = [x.cpu() for x in on_gpu[0]]
        held = [decode(m) if bits == 8 else tuple(t.clone() for t in m) for m in moments]
        none = [None] * len(SIZES)
        dev.adamw_step(on_gpu[0], on_gpu[1], [x.cuda() for x in grads], none, step=k, seeds=seeds, eps=eps, **HYPER)
        ref.adamw_step(p, moments, grads, none, step=k, seeds=seeds, eps=eps, **HYPER)
        for i in range(len(SIZES)):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(on_gpu[1][i], moments[i]))
            m = held[i][0] * b1 + grads[i] * (1 - b1)
            v = held[i][1] * b2 + grads[i] * (1 - b2) * grads[i]
            assert (v > 0).all() and (v < 2.0 ** -126).any()
            up = lr / (1 - b1 ** k) * m.double() / (v.double().sqrt() / math.sqrt(1 - b2 ** k) + eps)
            want = old[i].double() * (1 - lr * HYPER["weight_decay"]) - up
            got = on_gpu[0][i].cpu().double()
            # the quotient and the root to 2^-22 each, their factors in fp32, one rounding of p
            assert ((got - want).abs() <= 2.0 ** -23 * (old[i].double().abs() + want.abs()) + 2.0 ** -19 * up.abs()).all()
