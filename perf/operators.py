"""Operators of a training step around the transformer block, on their own: norms of the query and key heads with the rotation
in the same pass, the scaled token embedding with a gradient summed token by token, and AdamW over lists of tensors with its
moments in 32 bits or 8.

A case is a dict of plain values; `kind` says which operator:

* ``qk_fwd``   `qk_norm_rope_fwd` on the packed projection [B S, (Hq + 2 Hkv) D]: into a new tensor (``keep``: the backward pass
  needs the raw one) or in place.
* ``qk_bwd``   `qk_norm_rope_bwd`, in place on the packed gradient, the weight gradients added to their slots.
* ``emb_fwd``  `embedding_fwd` with ``scale`` (and learned positions where ``positions``).
* ``emb_bwd``  `embedding_bwd` with ``scale``, by token.
* ``adamw``    one `adamw_step` over a list of ``count`` tensors of ``numel`` elements and ``others`` of ``other_numel``, moments in
  ``bits`` bits.

The moments in 8 bits are the leading bits of the fp32 value (exponent and three bits of mantissa), counted from the block's
largest, and a sign for the first one; blocks have 256 elements.  What is rounded away is dithered with 16 bits of a hash of
the tensor's seed and the element's position.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 256


# ---------------------------------------------------------------------------------------------------------------- cases
def _case(**values):
    return {k: v for k, v in values.items() if v is not None}


def _qk(name, backward, batch, seq, q_heads, kv_heads, width, keep=True, reduce="float32", rope=True):
    return _case(name=name, kind="qk_bwd" if backward else "qk_fwd", batch=batch, seq=seq, q_heads=q_heads,
                 kv_heads=kv_heads, width=width, keep=keep, reduce=reduce, rope=rope)


def _emb(name, backward, batch, seq, vocab, hidden, spread, reduce="float32", positions=False):
    return _case(name=name, kind="emb_bwd" if backward else "emb_fwd", batch=batch, seq=seq, vocab=vocab,
                 hidden=hidden, spread=spread, reduce=reduce, positions=positions)


def _adamw(name, bits, count, numel, others, other_numel, reduce, step, decay):
    return _case(name=name, kind="adamw", bits=bits, count=count, numel=numel, others=others,
                 other_numel=other_numel, reduce=reduce, step=step, decay=decay)


def listed():
    return [
        # a block of the tiny decoder in a test or debugging job: 2 sequences of 128 tokens, a few microseconds of work
        _qk("qk_fwd_tiny", False, 2, 128, 8, 8, 64),
        # the forward pass of a schedule that recomputes (nothing kept), grouped heads of 64, an odd sequence length
        _qk("qk_fwd_1b_in_place", False, 2, 2047, 32, 8, 64, keep=False),
        # two long sequences through a 7B block with grouped heads, the raw projection kept for the backward pass
        _qk("qk_fwd_7b_gqa", False, 2, 8192, 32, 8, 128),
        _qk("qk_bwd_tiny", True, 2, 128, 8, 8, 64, reduce="bfloat16"),
        # two microbatches' worth of a 7B block, as many key heads as query heads, fp32 gradient bucket
        _qk("qk_bwd_7b", True, 2, 4096, 32, 32, 128),
        # one microbatch of a small GPT with learned positions
        _emb("emb_fwd_small", False, 2, 127, 1024, 256, "uniform", positions=True),
        # a global batch's share of one GPU, the 128k vocabulary, ids as text has them
        _emb("emb_fwd_1b", False, 8, 4096, 128256, 2048, "text"),
        # a debugging job's gradient: random ids into a bf16 bucket
        _emb("emb_bwd_tiny", True, 2, 128, 32000, 512, "uniform", reduce="bfloat16"),
        # 7B, four sequences, a fifth of all tokens one padding id and the rest as text has them
        _emb("emb_bwd_7b", True, 4, 4096, 32000, 4096, "padded"),
        # every parameter tensor of a toy model: launch-bound
        _adamw("adamw32_toy", 32, 4, 788736, 2, 327936, "float32", 1, 0.01),
        # the units of a 125M model, bf16 gradients
        _adamw("adamw32_125m", 32, 12, 7087872, 2, 39385344, "bfloat16", 1000, 0.1),
        # eight blocks of a 1B model, moments in 8 bits
        _adamw("adamw8_1b", 8, 8, 60821504, 1, 1000065, "float32", 250, 0.1),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["qk_fwd", "qk_bwd", "emb_fwd", "emb_bwd", "adamw", "adamw"])
    reduce = rng.choice(["float32", "bfloat16"])
    if kind.startswith("qk"):
        width = rng.choice([64, 64, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 3, 4, 8])
        q = kv * rng.choice([1, 2, 3, 4])
        batch = rng.choice([1, 2, 3])
        most = 16384 * 48 * 128 // ((q + 2 * kv) * width * batch)
        return _qk(None, kind == "qk_bwd", batch, log(1, min(16384, most)), q, kv, width, rng.random() < 0.6, reduce,
                   rng.random() < 0.8)
    if kind.startswith("emb"):
        hidden = 8 * log(8, 640)
        vocab = log(200, 130000)
        vocab = min(vocab, (1 << 28) // hidden)
        batch = rng.choice([1, 2, 3, 4])
        seq = log(1, min(16384, 50_000_000 // (hidden * batch)))
        return _emb(None, kind == "emb_bwd", batch, seq, vocab, hidden, rng.choice(["uniform", "text", "padded"]), reduce,
                    rng.random() < 0.3)
    count = rng.choice([1, 2, 5, 17, 70])
    numel = log(1000, 250_000_000 // count)
    return _adamw(None, rng.choice([8, 32]), count, numel, rng.choice([0, 1, 3]), log(1, 200_000), reduce, log(1, 10000),
                  rng.choice([0.0, 0.1]))


def work(case):
    c = case
    g = 4 if c.get("reduce") == "float32" else 2
    if c["kind"].startswith("qk"):
        T, qk, v, d = c["batch"] * c["seq"], c["q_heads"] + c["kv_heads"], c["kv_heads"], c["width"]
        table = min(c["seq"], T) * d * 4 if c["rope"] else 0
        if c["kind"] == "qk_bwd":
            return {"bytes": 3 * T * qk * d * 2 + T * qk * 4 + table + 4 * d * (1 + g), "flops": 16 * T * qk * d}
        kept = 2 * T * v * d * 2 + T * qk * 4 if c["keep"] else 0
        return {"bytes": 2 * T * qk * d * 2 + kept + table + 4 * d, "flops": 9 * T * qk * d}
    if c["kind"].startswith("emb"):
        T, H = c["batch"] * c["seq"], c["hidden"]
        p = _shares(c)
        distinct = float((1 - (1 - p) ** T).sum())
        if c["kind"] == "emb_fwd":
            pos = c["seq"] * H * 2 if c["positions"] else 0
            return {"bytes": int(8 * T + distinct * H * 2 + T * H * 2 + pos), "flops": 2 * T * H}
        pos = 2 * c["seq"] * H * g if c["positions"] else 0
        return {"bytes": int(8 * T + T * H * 2 + distinct * H * 2 * g + pos), "flops": 2 * T * H}
    n = c["count"] * c["numel"] + c["others"] * c["other_numel"]
    moments = 16 if c["bits"] == 32 else 4 + 4      # 8 bits: the codes, and the values that `run` returns
    return {"bytes": n * (8 + moments + g + 2), "flops": 16 * n}


# --------------------------------------------------------------------------------------------------------------- inputs
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _shares(case):
    """How often each rank of the vocabulary occurs: evenly, or as words do in text (Zipf-Mandelbrot); "padded": one id has a fifth."""
    V = case["vocab"]
    if case["spread"] == "uniform":
        return torch.full((V,), 1.0 / V, dtype=torch.float64)
    p = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
    p = p / p.sum()
    if case["spread"] == "padded":
        p = p * 0.8
        p[-1] += 0.2
    return p


def _table(S, d, device):
    """Cosines and sines of a rotation by theta = 500000, angles in 64 bits."""
    inv = 500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d)
    a = torch.arange(S, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _codes(x, most):
    """What moments in 8 bits are held as, rounded down: (codes, base of each block).  x >= 0, fp32."""
    n = x.numel()
    u = torch.nn.functional.pad(x.view(torch.int32), (0, -n % BLOCK)).view(-1, BLOCK)
    base = ((u.amax(1) + 0xFFFFF >> 20) - most).clamp_(min=0)
    code = ((u >> 20) - base[:, None]).clamp_(min=0).view(-1)[:n]
    return code.to(torch.uint8), base.to(torch.int16)


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    st = {"case": dict(c)}
    if c["kind"].startswith("qk"):
        T, nq, nk, d = c["batch"] * c["seq"], c["q_heads"], c["kv_heads"], c["width"]
        st |= {"qkv": normal(T, (nq + 2 * nk) * d, scale=0.7), "wq": normal(d, scale=0.2) + 1, "wk": normal(d, scale=0.2) + 1,
               "cs": _table(c["seq"], d, dev) if c["rope"] else None, "eps": 1e-5}
        if c["kind"] == "qk_bwd":
            x = st["qkv"][:, :(nq + nk) * d].float().view(T, nq + nk, d)
            gdt = _DTYPES[c["reduce"]]
            st |= {"rstd": torch.rsqrt(x.square().mean(-1) + st["eps"]), "dqkv": normal(T, (nq + 2 * nk) * d, scale=0.01),
                   "gwq": normal(d, scale=0.1, dtype=gdt), "gwk": normal(d, scale=0.1, dtype=gdt)}
    elif c["kind"].startswith("emb"):
        B, S, V, H = c["batch"], c["seq"], c["vocab"], c["hidden"]
        rank = torch.searchsorted(_shares(c).cumsum(0).to(dev), torch.rand(B, S, generator=gen, device=dev, dtype=torch.float64))
        ids = torch.randperm(V, generator=gen, device=dev)[rank.clamp_(max=V - 1)]
        st |= {"ids": ids.view(-1), "S": S, "scale": math.sqrt(H)}
        if c["kind"] == "emb_fwd":
            st |= {"table": normal(V, H, scale=0.02), "pos": normal(S, H, scale=0.02) if c["positions"] else None}
        else:
            gdt = _DTYPES[c["reduce"]]
            st |= {"dout": normal(B * S, H, scale=0.01), "gtable": normal(V, H, scale=0.01, dtype=gdt),
                   "gpos": normal(S, H, scale=0.01, dtype=gdt) if c["positions"] else None}
    else:
        sizes = [c["numel"]] * c["count"] + [c["other_numel"]] * c["others"]
        starts, total = [], 0
        for n in sizes:         # the tensors of a model, one after another, each at the start of a block
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        gdt = _DTYPES[c["reduce"]]
        flat = {"p": normal(total, scale=0.02, dtype=torch.float32), "p16": torch.zeros(total, dtype=torch.bfloat16, device=dev)}
        flat["g"] = normal(total, dtype=torch.float32).exp_().mul_(normal(total, scale=1e-3, dtype=torch.float32)).to(gdt)
        m, v = normal(total, scale=3e-5, dtype=torch.float32), normal(total, scale=1e-4, dtype=torch.float32).square_()
        used = torch.cat([t for n in sizes for t in (torch.ones(n, device=dev), torch.zeros(-n % BLOCK, device=dev))])
        used *= c["step"] > 1
        m *= used
        v *= used
        if c["bits"] == 8:
            code, flat["mb"] = _codes(m.abs(), 127)
            flat["m"] = code | (m < 0).to(torch.uint8) * 128
            flat["v"], flat["vb"] = _codes(v, 255)
        else:
            flat |= {"m": m, "v": v}

        def views(k):
            if k in ("mb", "vb"):
                return [flat[k][o // BLOCK:-(-(o + n) // BLOCK)] for o, n in zip(starts, sizes)]
            return [flat[k][o:o + n] for o, n in zip(starts, sizes)]

        moments = ("m", "mb", "v", "vb") if c["bits"] == 8 else ("m", "v")
        st |= {"flat": flat, "p": views("p"), "p16": views("p16"), "g": views("g"),
               "moments": list(zip(*(views(k) for k in moments))), "seeds": [(int(seed) * 7919 + 104729 * i) % 2 ** 32 for i in range(len(sizes))],
               "hyper": {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": c["decay"], "step": c["step"],
                         "grad_scale": 0.125}}
    return st


# ----------------------------------------------------------------------------------------------------------- plain forms
def _values(code, base):
    """What the codes of a tensor stand for, without their sign."""
    c = code.to(torch.int32)
    b = base.to(torch.int32).repeat_interleave(BLOCK)[:c.numel()]
    return torch.where(c > 0, (c + b) << 20, c).view(torch.float32)


def _signed(code, base):
    x = _values(code & 127, base)
    return torch.where(code > 127, -x, x)


def _dither(n, seed, device):
    x = torch.arange(-(-n // 2), dtype=torch.int64, device=device) * 0x9E3779B1 + seed & 0xFFFFFFFF
    x = (x ^ x >> 15) * 0x6A09E667 & 0xFFFFFFFF
    x = (x ^ x >> 13) * 0xBB67AE85 & 0xFFFFFFFF
    x = x ^ x >> 16
    return (torch.stack([x & 0xFFFF, x >> 16], 1) << 4 | 8).view(-1)[:n].to(torch.int32)


def _round8(x, dither, most, least):
    """Codes and bases of x >= 0; `least` is the code of the smallest values that are not 0."""
    n = x.numel()
    bits = x.view(torch.int32).clamp(max=0x7FE00000)
    u = torch.nn.functional.pad(bits, (0, -n % BLOCK)).view(-1, BLOCK)
    base = ((u.amax(1) + 0xFFFFF >> 20) - most).clamp_(min=0)
    code = (bits + dither >> 20) - base.repeat_interleave(BLOCK)[:n]
    code = torch.where(bits > 0, code.clamp_(min=least), 0)
    return code.to(torch.uint8), base.to(torch.int16)


def _qk_parts(st):
    c = st["case"]
    T, nq, nk, d = st["qkv"].shape[0], c["q_heads"], c["kv_heads"], c["width"]
    x = st["qkv"][:, :(nq + nk) * d].float().view(T, nq + nk, d)
    w = torch.cat([st["wq"].float().expand(nq, d), st["wk"].float().expand(nk, d)])
    return x, w, (nq + nk) * d


def _rotate(x, cs, S, sign):
    if cs is None:
        return x
    T, h = x.shape[0], x.shape[2] // 2
    at = torch.arange(T, device=x.device) % S
    co, si = cs[at, None, :h], cs[at, None, h:] * sign
    return torch.cat([x[..., :h] * co - x[..., h:] * si, x[..., h:] * co + x[..., :h] * si], -1)


def _plain_qk_fwd(st):
    c, (x, w, cut) = st["case"], _qk_parts(st)
    rstd = 1.0 / torch.sqrt((x * x).mean(-1) + st["eps"])
    y = _rotate(x * rstd[..., None] * w, st["cs"], c["seq"], 1.0).reshape(x.shape[0], cut)
    out = st["qkv"].clone() if c["keep"] else st["qkv"]
    out[:, :cut] = y.to(out.dtype)
    return {"qkv": out, "rstd": rstd} if c["keep"] else {"qkv": out}


def _plain_qk_bwd(st):
    c, (x, w, cut) = st["case"], _qk_parts(st)
    nq = c["q_heads"]
    g = _rotate(st["dqkv"][:, :cut].float().view(x.shape), st["cs"], c["seq"], -1.0)
    xh = x * st["rstd"][..., None]
    dw = (g * xh).sum(0)
    wg = w * g
    dx = st["rstd"][..., None] * (wg - xh * (wg * xh).mean(-1, keepdim=True))
    st["dqkv"][:, :cut] = dx.reshape(x.shape[0], cut).to(st["dqkv"].dtype)
    st["gwq"].copy_(st["gwq"].float() + dw[:nq].sum(0))
    st["gwk"].copy_(st["gwk"].float() + dw[nq:].sum(0))
    return {k: st[k] for k in ("dqkv", "gwq", "gwk")}


def _plain_emb_fwd(st):
    y = st["table"][st["ids"]].float() * st["scale"]
    if st["pos"] is not None:
        y = y + st["pos"].float().repeat(y.shape[0] // st["S"], 1)
    return y.to(st["table"].dtype)


def _plain_emb_bwd(st):
    d = st["dout"].float()
    st["gtable"].copy_(st["gtable"].float().index_add_(0, st["ids"], d * st["scale"]))
    if st["gpos"] is not None:
        st["gpos"].copy_(st["gpos"].float() + d.view(-1, st["S"], d.shape[1]).sum(0))
        return {"gtable": st["gtable"], "gpos": st["gpos"]}
    return {"gtable": st["gtable"]}


def _plain_adamw_one(st, i):
    h, bits, moments = st["hyper"], st["case"]["bits"], st["moments"][i]
    p, g = st["p"][i], st["g"][i].float() * h["grad_scale"]
    m, v = moments if bits == 32 else (_signed(*moments[:2]), _values(*moments[2:]))
    m = m * h["beta1"] + g * (1 - h["beta1"])
    v = v * h["beta2"] + g * (1 - h["beta2"]) * g
    denom = torch.sqrt(v) * (1 / math.sqrt(1 - h["beta2"] ** h["step"])) + h["eps"]
    p.copy_(p * (1 - h["lr"] * h["weight_decay"]) - m / denom * (h["lr"] / (1 - h["beta1"] ** h["step"])))
    st["p16"][i].copy_(p)
    if bits == 8:
        dither = _dither(p.numel(), st["seeds"][i], p.device)
        code, base = _round8(m.abs(), dither, 127, 0)
        new = (code | torch.signbit(m).to(torch.uint8) * 128, base, *_round8(v, dither, 255, 1))
    else:
        new = m, v
    return [old.copy_(x) for old, x in zip(moments, new)]


def _plain_adamw(st):
    f = st["flat"]
    [_plain_adamw_one(st, i) for i in range(len(st["p"]))]
    if st["case"]["bits"] == 32:
        return {"p": f["p"], "p16": f["p16"], "m": f["m"], "v": f["v"]}
    # moments in 8 bits as the values they stand for, whose four leading bits bf16 holds
    return {"p": f["p"], "p16": f["p16"], "m": _signed(f["m"], f["mb"]).bfloat16(), "v": _values(f["v"], f["vb"]).bfloat16()}


# -------------------------------------------------------------------------------------------------------------------- run
def run(state):
    if own:
        return _run_own(state)
    plain = {"qk_fwd": _plain_qk_fwd, "qk_bwd": _plain_qk_bwd, "emb_fwd": _plain_emb_fwd, "emb_bwd": _plain_emb_bwd,
             "adamw": _plain_adamw}
    return plain[state["case"]["kind"]](state)


def _run_own(st):
    from zorse_b200.ops.api import get_ops

    ops, c = get_ops("sm100"), st["case"]
    if c["kind"] == "qk_fwd":
        out, rstd = ops.qk_norm_rope_fwd(st["qkv"], st["wq"], st["wk"], st["cs"], c["seq"], c["q_heads"], c["kv_heads"], c["width"],
                                         st["eps"], keep=c["keep"])
        return {"qkv": out, "rstd": rstd} if c["keep"] else {"qkv": out}
    if c["kind"] == "qk_bwd":
        ops.qk_norm_rope_bwd(st["dqkv"], st["qkv"], st["wq"], st["wk"], st["rstd"], st["cs"], c["seq"], c["q_heads"],
                             c["kv_heads"], c["width"], st["gwq"], st["gwk"])
        return {k: st[k] for k in ("dqkv", "gwq", "gwk")}
    if c["kind"] == "emb_fwd":
        return ops.embedding_fwd(st["ids"], st["table"], st["pos"], st["S"], 0, scale=st["scale"])
    if c["kind"] == "emb_bwd":
        ops.embedding_bwd(st["ids"], st["dout"], st["gtable"], st["gpos"], st["S"], 0, scale=st["scale"], by_token=True)
        return {"gtable": st["gtable"]} if st["gpos"] is None else {"gtable": st["gtable"], "gpos": st["gpos"]}
    f = st["flat"]
    ops.adamw_step(st["p"], st["moments"], st["g"], st["p16"], seeds=st["seeds"] if c["bits"] == 8 else None, **st["hyper"])
    if c["bits"] == 32:
        return {"p": f["p"], "p16": f["p16"], "m": f["m"], "v": f["v"]}
    m, v = ops.moment_values((f["m"], f["mb"], f["v"], f["vb"]), torch.bfloat16)
    return {"p": f["p"], "p16": f["p16"], "m": m, "v": v}


# ---------------------------------------------------------------------------------------------------------- 64-bit answers
def _leading(x):
    """A value's place on the scale of fp32 patterns (2^49 to a code), from its 64-bit pattern."""
    return (x.view(torch.int64) - (896 << 52)).clamp_(min=0)


def _stands_for(u):
    """The value of a code counted from zero: exponent and three bits of mantissa."""
    return torch.where(u >= 8, (u + 896 * 8) << 49, 0).view(torch.float64)


def _per_block(x, n):
    return x.to(torch.int64)[:, None].expand(-1, BLOCK).reshape(-1)[:n]


def _read(code, base):
    code = code.to(torch.int64)
    return torch.where(code == 0, 0.0, _stands_for(code + _per_block(base, code.numel())))


def _held(x, noise, most, least):
    n = x.numel()
    y = _leading(x)
    top = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.int64, device=x.device)
    top[:n] = y
    base = (-(-top.view(-1, BLOCK).amax(1) // 2 ** 49) - most).clamp_(min=0)
    u = ((y + noise * 2 ** 33 + 2 ** 32) >> 49) - _per_block(base, n)
    u = torch.where(x == 0, 0, u.clamp_(min=least))
    return torch.where(u == 0, 0.0, _stands_for(u + _per_block(base, n)))


def _noise(n, seed, device):
    """Half of the hash of each pair of positions, in arithmetic modulo 2^32 on signed words."""
    def word(x):
        return torch.tensor(x - 2 ** 32 if x >= 2 ** 31 else x, dtype=torch.int32, device=device)

    def fold(x, k):
        return x ^ (x >> k & (1 << 32 - k) - 1)

    at = torch.arange(n, device=device)
    x = (at >> 1).to(torch.int32) * word(0x9E3779B1) + word(seed)
    x = fold(fold(fold(x, 15) * word(0x6A09E667), 13) * word(0xBB67AE85), 16)
    return (x >> (at & 1).to(torch.int32) * 16).to(torch.int64) & 0xFFFF


def _exact_adamw(st):
    h, bits, f = st["hyper"], st["case"]["bits"], st["flat"]
    out = {k: f[k].double() for k in ("p", "p16")} | {k: torch.zeros_like(f["p"], dtype=torch.float64) for k in ("m", "v")}
    if bits == 32:
        out |= {k: f[k].double() for k in ("m", "v")}
    else:
        out["m"] = _read(f["m"] % 128, f["mb"]) * (1.0 - 2.0 * (f["m"] // 128))
        out["v"] = _read(f["v"], f["vb"])
    for i, part in enumerate(st["p"]):
        n, o = part.numel(), part.storage_offset()
        p, p16, m, v = (out[k][o:o + n] for k in ("p", "p16", "m", "v"))
        g = st["g"][i].double() * h["grad_scale"]
        m += (1 - h["beta1"]) * (g - m)
        v += (1 - h["beta2"]) * (g * g - v)
        mean, root = m / (1 - h["beta1"] ** h["step"]), (v / (1 - h["beta2"] ** h["step"])).sqrt_()
        p -= h["lr"] * (h["weight_decay"] * p + mean / (root + h["eps"]))
        p16.copy_(p)
        del mean, root, g
        if bits == 8:
            noise = _noise(n, st["seeds"][i], p.device)
            m.copy_(torch.copysign(_held(m.abs(), noise, 127, 0), m))
            v.copy_(_held(v.contiguous(), noise, 255, 1))
    return out


def exact(case, seed):
    """What `run` returns for the inputs of this seed, in 64 bits."""
    st = prepare(case, seed)
    c = case
    if c["kind"] == "adamw":
        return _exact_adamw(st)
    if c["kind"].startswith("emb"):
        ids, S, B = st["ids"], c["seq"], c["batch"]
        if c["kind"] == "emb_fwd":
            y = torch.nn.functional.embedding(ids, st["table"]).double().mul_(st["scale"]).view(B, S, -1)
            return (y if st["pos"] is None else y + st["pos"].double()).view(B * S, -1)
        dout = st["dout"].double()
        sums = torch.zeros(st["gtable"].shape, dtype=torch.float64, device=dout.device)
        sums.scatter_add_(0, ids[:, None].expand(-1, c["hidden"]), dout)
        out = {"gtable": sums.mul_(st["scale"]).add_(st["gtable"])}
        if st["gpos"] is not None:
            out["gpos"] = st["gpos"].double() + dout.view(B, S, -1).sum(0)
        return out
    nq, nk, d, S, B = c["q_heads"], c["kv_heads"], c["width"], c["seq"], c["batch"]
    h = d // 2
    turn = torch.ones(S, h, dtype=torch.complex128, device=st["qkv"].device)
    if c["rope"]:
        turn = torch.complex(st["cs"][:, :h].double(), st["cs"][:, h:].double())
    turn = turn.view(1, S, 1, h)
    out = (st["qkv"] if c["kind"] == "qk_fwd" else st["dqkv"]).double()
    rstds, slots = [], []
    for at, n, w in ((0, nq, st["wq"].double()), (nq * d, nk, st["wk"].double())):
        x = st["qkv"][:, at:at + n * d].double().view(B, S, n, d)
        if c["kind"] == "qk_fwd":
            rstd = (x.square().mean(-1, keepdim=True) + st["eps"]) ** -0.5
            y = x * rstd * w
            z = torch.complex(y[..., :h].contiguous(), y[..., h:].contiguous()) * turn
            out[:, at:at + n * d] = torch.cat([z.real, z.imag], -1).view(B * S, -1)
            rstds.append(rstd.view(B * S, n))
        else:
            rstd = st["rstd"][:, at // d:at // d + n].double().view(B, S, n, 1)
            y = out[:, at:at + n * d].view(B, S, n, d)
            z = torch.complex(y[..., :h].contiguous(), y[..., h:].contiguous()) * turn.conj()
            g = torch.cat([z.real, z.imag], -1)
            slots.append((g * x * rstd).sum((0, 1, 2)))
            along = (g * w * x).mean(-1, keepdim=True) * rstd ** 2
            out[:, at:at + n * d] = ((g * w - x * along) * rstd).view(B * S, -1)
    if c["kind"] == "qk_bwd":
        return {"dqkv": out, "gwq": st["gwq"].double() + slots[0], "gwk": st["gwk"].double() + slots[1]}
    return {"qkv": out, "rstd": torch.cat(rstds, 1)} if c["keep"] else {"qkv": out}
