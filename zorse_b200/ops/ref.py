"""Pure-PyTorch restatement of every op (runs on CPU, any dtype).

This is the oracle the sm_100a kernels are tested against and the compute backend of the
CPU/gloo configuration.  Shapes follow the packed layouts the CUDA kernels use:
`qkv` is `[T, (Hq + 2*Hkv) * D]` (query heads, key heads, value heads).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F

from .moments import decode, dither, encode


def linear(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None) -> torch.Tensor:
    y = x @ w.t()
    return y if b is None else y + b


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * rstd * w.float()).to(x.dtype)


def layernorm(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    xf = x.float()
    mu = xf.mean(-1, keepdim=True)
    var = (xf - mu).pow(2).mean(-1, keepdim=True)
    y = (xf - mu) * torch.rsqrt(var + eps) * w.float()
    if b is not None:
        y = y + b.float()
    return y.to(x.dtype)


def rope_table(S: int, d: int, theta: float, device=None) -> torch.Tensor:
    """[S, d] fp32: cos (d/2) | sin (d/2) for positions 0..S-1 (rotate-half convention)."""
    inv = 1.0 / (theta ** (torch.arange(0, d, 2, dtype=torch.float64, device=device) / d))
    ang = torch.arange(S, dtype=torch.float64, device=device)[:, None] * inv[None, :]
    return torch.cat([ang.cos(), ang.sin()], dim=-1).float()


def rope(qkv: torch.Tensor, cs: torch.Tensor, S: int, nheads: int, d: int, backward: bool = False) -> torch.Tensor:
    """Rotates heads [0, nheads) of packed qkv [T, width]; returns a new tensor."""
    T = qkv.shape[0]
    out = qkv.clone()
    x = qkv[:, : nheads * d].float().reshape(T, nheads, d)
    pos = torch.arange(T, device=qkv.device) % S
    cos = cs[pos, : d // 2][:, None, :]
    sin = cs[pos, d // 2:][:, None, :]
    if backward:
        sin = -sin
    a, b = x[..., : d // 2], x[..., d // 2:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    out[:, : nheads * d] = y.reshape(T, nheads * d).to(qkv.dtype)
    return out


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    F_ = gu.shape[-1] // 2
    g, u = gu[..., :F_].float(), gu[..., F_:].float()
    return (F.silu(g) * u).to(gu.dtype)


def activation(x: torch.Tensor, kind: str) -> torch.Tensor:
    xf = x.float()
    if kind == "relu":
        y = F.relu(xf)
    elif kind == "gelu_erf":
        y = F.gelu(xf)
    else:
        y = F.gelu(xf, approximate="tanh")
    return y.to(x.dtype)


def attention(qkv: torch.Tensor, B: int, S: int, Hq: int, Hkv: int, D: int, causal: bool = True,
              window: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """Explicit masked-softmax attention in fp32. Returns [B*S, Hq*D] in qkv's dtype."""
    sc = 1.0 / math.sqrt(D) if scale is None else scale
    x = qkv.float().reshape(B, S, Hq + 2 * Hkv, D)
    q = x[:, :, :Hq].permute(0, 2, 1, 3)
    k = x[:, :, Hq:Hq + Hkv].permute(0, 2, 1, 3)
    v = x[:, :, Hq + Hkv:].permute(0, 2, 1, 3)
    rep = Hq // Hkv
    k = k.repeat_interleave(rep, dim=1)
    v = v.repeat_interleave(rep, dim=1)
    s = (q @ k.transpose(-1, -2)) * sc
    i = torch.arange(S, device=qkv.device)[:, None]
    j = torch.arange(S, device=qkv.device)[None, :]
    mask = torch.ones(S, S, dtype=torch.bool, device=qkv.device)
    if causal:
        mask &= j <= i
    if window and window > 0:
        mask &= (i - j) < window
    s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    o = p @ v
    return o.permute(0, 2, 1, 3).reshape(B * S, Hq * D).to(qkv.dtype)


def _turn(x, cs, S: int, sign: float):
    """Heads x [T, n, d] rotated by the angles of row t mod S of cs; None: as they are."""
    if cs is None:
        return x
    h = x.shape[2] // 2
    pos = torch.arange(x.shape[0], device=x.device) % S
    cos, sin = cs[pos, None, :h], sign * cs[pos, None, h:]
    return torch.cat([x[..., :h] * cos - x[..., h:] * sin, x[..., h:] * cos + x[..., :h] * sin], dim=-1)


def _heads_and_weights(qkv, wq, wk, nq: int, nk: int, d: int):
    x = qkv[:, : (nq + nk) * d].float().reshape(qkv.shape[0], nq + nk, d)
    return x, torch.cat([wq.float().expand(nq, d), wk.float().expand(nk, d)])


def qk_norm_rope(qkv, wq, wk, cs, S: int, nq: int, nk: int, d: int, eps: float):
    """(qkv with query and key heads RMS-normalised and rotated, 1 / rms of these heads [T, nq + nk])."""
    x, w = _heads_and_weights(qkv, wq, wk, nq, nk, d)
    rstd = torch.rsqrt(x.pow(2).mean(-1) + eps)
    y = _turn(x * rstd[..., None] * w, cs, S, 1.0).reshape(qkv.shape[0], (nq + nk) * d)
    return torch.cat([y.to(qkv.dtype), qkv[:, (nq + nk) * d:]], dim=1), rstd


def qk_norm_rope_bwd(dqkv, qkv, wq, wk, rstd, cs, S: int, nq: int, nk: int, d: int):
    """fp32 gradients of the query and key heads [T, (nq + nk) d], of wq and of wk."""
    x, w = _heads_and_weights(qkv, wq, wk, nq, nk, d)
    g = _turn(dqkv[:, : (nq + nk) * d].float().reshape(x.shape), cs, S, -1.0)
    xh = x * rstd[..., None]
    dw = (g * xh).sum(0)
    dx = rstd[..., None] * (w * g - xh * (w * g * xh).mean(-1, keepdim=True))
    return dx.reshape(qkv.shape[0], (nq + nk) * d), dw[:nq].sum(0), dw[nq:].sum(0)


def cross_entropy_rows(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    return F.cross_entropy(logits.float(), targets, reduction="none")


def embedding(ids: torch.Tensor, table: torch.Tensor, pos_table: Optional[torch.Tensor] = None, S: int = 1,
              pos_offset: int = 0, scale: float = 1.0) -> torch.Tensor:
    out = table[ids.reshape(-1)]
    if scale != 1.0:
        out = out.float() * scale
    if pos_table is not None:
        pos = torch.arange(ids.numel(), device=ids.device) % S + pos_offset
        out = out + pos_table[pos]
    return out.to(table.dtype)


def adam_step(p, m, v, g, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    """In-place fp32 Adam with torch.optim.Adam arithmetic."""
    g = g.float() * grad_scale
    if weight_decay:
        g = g + weight_decay * p
    m.mul_(beta1).add_(g, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    denom = v.sqrt() / math.sqrt(bc2) + eps
    p.addcdiv_(m, denom, value=-lr / bc1)


def adamw_step(p, moments, g, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0, seed=0):
    """In-place AdamW (decoupled decay) on one fp32 tensor; moments: (m, v) in fp32, or `Moments8`, rounded with the dither of `seed`.
    Every operation on the moments rounds by itself, as in the kernel."""
    held = len(moments) == 4
    m, v = decode(moments) if held else (t.reshape(-1) for t in moments)
    x, g = p.view(-1), g.reshape(-1).float() * grad_scale
    m = m * beta1 + g * (1 - beta1)
    v = v * beta2 + g * (1 - beta2) * g
    update = m / (v.sqrt() / math.sqrt(1 - beta2 ** step) + eps)
    x.copy_(x * (1 - lr * weight_decay) - lr / (1 - beta1 ** step) * update)
    for old, new in zip(moments, encode(m, v, dither(x.numel(), seed, x.device)) if held else (m, v)):
        old.view(-1).copy_(new)
