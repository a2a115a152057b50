"""Bounds as tight as the arithmetic allows: the sums of the embedding gradient by token, and the mean of what the dither holds."""
import pytest
import torch

from zorse_b200.ops.api import get_ops
from zorse_b200.ops.moments import decode, dither, dither_seed, encode
from test_embedding_by_token import SHAPES, _ids, _normal


def test_the_dither_holds_the_value_on_average_cpu():
    """A value f of the way from one code to the next is held as the upper one with probability f: a standard error of
    sqrt(f (1 - f) / seeds) steps.  The dither has 16 bits, so f is known to 2^-17."""
    x = torch.tensor([1.03, 1.0001, 3.7, 0.9, 1.0625, 1.999])
    seeds = 1 << 14
    held = torch.stack([decode(encode(x, x, dither(6, dither_seed(s, 5))))[0] for s in range(seeds)]).double()
    width = 2.0 ** (torch.floor(torch.log2(x.double())) - 3)
    f = (x.double() / width) % 1
    low = x.double() - f * width
    assert ((held == low) | (held == low + width)).all()
    assert ((held.mean(0) - x.double()).abs() <= (6 * (f * (1 - f) / seeds).sqrt() + 2.0 ** -16) * width).all()


def _chain(ids, V):
    """Additions that a term of a row goes through at most, for each id: 32 rows of a piece one behind the other; of a run over
    several pieces of four rows at least, up to 17 parts or an eighth of all, in one kernel for few tokens an eighth of the rows;
    then eight partial sums, the factor and the old value."""
    n = torch.bincount(ids, minlength=V).double()
    pieces = (n / 4).ceil() + 1
    return torch.maximum(32 + torch.maximum(torch.tensor(17.0), (pieces / 8).ceil()), (n / 8).ceil()) + 10


@pytest.mark.gpu
@pytest.mark.parametrize("T,S,V,H", SHAPES)
@pytest.mark.parametrize("kind", ["any", "one", "hot", "few", "runs"])
@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
def test_sums_by_token(T, S, V, H, kind, grads):
    ids, dout, old = _ids(T, V, kind), _normal(T, H), _normal(V, H, seed=1, dtype=grads)
    table = old.cuda()
    scale = 1.7
    get_ops("sm100").embedding_bwd(ids.cuda(), dout.cuda(), table, scale=scale, by_token=True)
    d = dout.double() * float(torch.tensor(scale))           # the factor as the kernel has it
    want, size = old.double().index_add(0, ids, d), old.double().abs().index_add(0, ids, d.abs())
    half = torch.finfo(grads).eps / 2
    bound = half * want.abs() + (1 + half) * 2.0 ** -24 * _chain(ids, V)[:, None] * size
    got = table.cpu().double()
    assert ((got - want).abs() <= bound).all()
    # A test of the test: a sum with its largest term missing is out of bounds.  n terms of mean size 1.7 x 0.8 have a bound of about
    # (n / 32 + 42) 2^-24 1.36 n, which the largest of them (above 5) exceeds up to n of some ten thousand; longer sums are counted
    # row by row in whole numbers elsewhere.
    at = int(torch.bincount(ids, minlength=V).argmax())
    terms = d[ids == at]
    if grads is torch.float32 and terms.shape[0] <= 8192:
        assert (terms.abs().max(0).values > bound[at]).any()
