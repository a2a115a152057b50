"""Adam's moments in 8 bits: what their codes mean (csrc/optim/adamw_list.cu has the step itself).

A value is held as the leading bits of its fp32 pattern, exponent and three bits of mantissa (`bits >> 20`), counted from a base
that a block of 256 values shares: m as its sign and 0 .. 127, v as 0 .. 255.  Code 0 is zero, and a v above zero keeps at
least code 1.  The base is such that the block's largest value fits, so m reaches 16 binades below it and v 32.  What is held
is exact in bf16 and in fp32, and encoding it again gives the same values.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

BLOCK = 256
_M_MOST, _V_MOST = 127, 255
_TOP = 0x7FE00000                       # NaNs, whatever their pattern, are held as this one


class Moments8(NamedTuple):
    """Codes [n] (uint8) and bases of the blocks (int16) of both moments."""
    m: torch.Tensor
    m_base: torch.Tensor
    v: torch.Tensor
    v_base: torch.Tensor

    @classmethod
    def zeros(cls, n: int, device=None) -> "Moments8":
        blocks = -(-n // BLOCK)
        return cls(*(torch.zeros(k, dtype=t, device=device)
                     for k, t in ((n, torch.uint8), (blocks, torch.int16), (n, torch.uint8), (blocks, torch.int16))))

    def load(self, m: torch.Tensor, v: torch.Tensor) -> None:
        """Takes over fp32 values, rounded to nearest."""
        for old, new in zip(self, encode(m, v)):
            old.copy_(new)


def _spread(base, n):
    return base.to(torch.int32).repeat_interleave(BLOCK)[:n]


def _decode(code, base):
    c = code.to(torch.int32)
    return torch.where(c > 0, (c + _spread(base, c.numel())) << 20, c).view(torch.float32)


def decode(moments) -> tuple[torch.Tensor, torch.Tensor]:
    """The fp32 values (m, v) that codes stand for."""
    code, m_base, v, v_base = moments
    m = _decode(code & 127, m_base)
    return torch.where(code > 127, -m, m), _decode(v, v_base)


def _encode(x, add, most, least):
    n = x.numel()
    bits = x.contiguous().view(torch.int32)
    bits = torch.where(torch.isnan(x), _TOP, bits)       # (a NaN may have its sign bit set, and be a negative number here)
    blocks = torch.nn.functional.pad(bits, (0, -n % BLOCK)).view(-1, BLOCK)
    base = ((blocks.amax(1) + 0xFFFFF >> 20) - most).clamp_(min=0)
    code = ((bits + add >> 20) - _spread(base, n)).clamp_(min=least)
    return torch.where(bits > 0, code, 0).to(torch.uint8), base.to(torch.int16)


def encode(m: torch.Tensor, v: torch.Tensor, add=0x80000) -> Moments8:
    """Codes of fp32 values; `add`: what goes to the patterns before they are cut (a half: to nearest; or `dither`)."""
    m, v = m.reshape(-1).float(), v.reshape(-1).float()
    code, base = _encode(m.abs(), add, _M_MOST, 0)
    return Moments8(code | torch.signbit(m).to(torch.uint8) << 7, base, *_encode(v, add, _V_MOST, 1))


_WORD = 0xFFFFFFFF


def _mix(x):
    x = (x ^ x >> 15) * 0x6A09E667 & _WORD
    x = (x ^ x >> 13) * 0xBB67AE85 & _WORD
    return x ^ x >> 16


def dither(n: int, seed: int, device=None) -> torch.Tensor:
    """What the step adds to the patterns of n elements: 16 bits of a hash of the seed and the pair of elements, below bit 20."""
    pair = torch.arange(-(-n // 2), dtype=torch.int64, device=device)
    x = _mix(pair * 0x9E3779B1 + (seed & _WORD) & _WORD)
    return (torch.stack([x & 0xFFFF, x >> 16], dim=1) << 4 | 8).view(-1)[:n].to(torch.int32)


def dither_seed(*parts: int) -> int:
    """A seed for `dither` from whole numbers (the job's seed, the tensor, the step)."""
    x = 0
    for p in parts:
        x = _mix(x * 0x9E3779B1 + (p & _WORD) + 1 & _WORD)
    return x
