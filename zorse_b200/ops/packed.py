"""Packed batches: sequences of different lengths, one after another, in one stream of T tokens (csrc/attn/packed.cu).

`PackedSequences` is made once for a batch and used by every layer.  Tokens behind the last sequence belong to none: attention gives
them zeros (and -inf for the log-sum-exp), and whatever they hold reaches nobody.  A NaN or an infinity in a sequence can reach its
neighbours in the batch: a weight of 0 times it is NaN.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

MOST_TOKENS = 65535 * 128
MOST_AXES = 4
PACK_SCAN = 4096      # sequences whose offsets every block of the plan looks at (csrc/attn/packed.cu)


class PackedSequences(NamedTuple):
    """tokens: T.  bounds [T rounded up to 256, 2]: begin and end of each token's sequence.  positions [T]: places within the sequences
    (0 for tokens of none).  The orders, of the kernels alone: a record for each tile, long sequences first."""
    tokens: int
    bounds: torch.Tensor
    positions: torch.Tensor
    order_pairs: Optional[torch.Tensor] = None
    order_tiles: Optional[torch.Tensor] = None
    order_keys: Optional[torch.Tensor] = None


def check_window(causal: bool, window: int) -> None:
    if window < 0 or (window and not causal):
        raise ValueError(f"window {window}: a positive one is for causal attention (0: none)")


def pack(offsets: torch.Tensor, T: int) -> PackedSequences:
    ends = offsets[1:].contiguous()
    total = int(offsets[-1]) if ends.numel() else 0
    if offsets.numel() < 1 or bool((offsets[1:] < offsets[:-1]).any()) or int(offsets[0]) != 0 or total > T:
        raise ValueError(f"offsets rise from 0 to at most {T} tokens")
    t = torch.arange(-(-T // 256) * 256, dtype=offsets.dtype, device=offsets.device)
    doc = torch.searchsorted(ends, t, right=True).clamp_(max=max(ends.numel() - 1, 0))
    inside = (t < total)[:, None]
    bounds = torch.stack([offsets[doc], ends[doc]], 1) if ends.numel() else torch.zeros(t.numel(), 2, dtype=torch.int32, device=t.device)
    bounds = torch.where(inside, bounds, torch.full_like(bounds, total)).to(torch.int32)
    return PackedSequences(T, bounds, torch.where(inside[:, 0], t - bounds[:, 0], 0).to(torch.int32)[:T])


def seen(packed: PackedSequences, causal: bool, window: int) -> torch.Tensor:
    """[T, T]: which keys (columns) a token (row) sees."""
    check_window(causal, window)
    T = packed.tokens
    lo, hi = packed.bounds[:T, 0, None], packed.bounds[:T, 1, None]
    t = torch.arange(T, dtype=torch.int32, device=lo.device)
    keys = (t >= lo) & (t < hi)
    if causal:
        keys &= t <= t[:, None]
    if window:
        keys &= t[:, None] - t < window
    return keys


def attention(qkv, packed: PackedSequences, Hq: int, Hkv: int, D: int, causal: bool = True, window: int = 0):
    """(out [T, Hq D] in qkv's type, lse [Hq, T]); at least fp32 inside."""
    T = packed.tokens
    inside = (packed.bounds[:T, 0] < packed.bounds[:T, 1])[:, None]
    x = torch.where(inside, qkv.to(torch.promote_types(qkv.dtype, torch.float32)), 0.0).reshape(T, Hq + 2 * Hkv, D).transpose(0, 1)
    rep = Hq // Hkv
    k, v = (x[Hq + i * Hkv:Hq + (i + 1) * Hkv].repeat_interleave(rep, dim=0) for i in (0, 1))
    alone = torch.eye(T, dtype=torch.bool, device=x.device) & ~inside      # (a row of nothing has no softmax)
    s = (x[:Hq] @ k.transpose(1, 2) / math.sqrt(D)).masked_fill(~(seen(packed, causal, window) | alone), -math.inf)
    o = torch.softmax(s, 2) @ v
    return o.transpose(0, 1).reshape(T, Hq * D).to(qkv.dtype), torch.where(inside[:, 0], torch.logsumexp(s, 2), -math.inf)


def rope_at(buf, cs, positions, nheads: int, d: int, sections=None, backward: bool = False):
    """Heads [0, nheads) of buf [T, width] turned by the rows `positions` [axes, T] (or [T]) of cs; returns a new tensor."""
    T, h = buf.shape[0], d // 2
    positions = positions.reshape(-1, T)
    sections = [h] if sections is None else list(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(buf.device)
    at = positions.long()[axis].t().clamp(0, cs.shape[0] - 1)
    cos, sin = cs[:, :h].gather(0, at)[:, None], cs[:, h:].gather(0, at)[:, None]
    x = buf[:, :nheads * d].to(torch.promote_types(buf.dtype, torch.float32)).reshape(T, nheads, d)
    a, b = x[..., :h], x[..., h:]
    sin = -sin if backward else sin
    out = buf.clone()
    out[:, :nheads * d] = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).reshape(T, nheads * d).to(buf.dtype)
    return out
