"""Operators of training on packed batches and of the Muon optimizer, on their own: attention over sequences of different lengths
that lie one after another in one batch, rotation of heads by given positions of one or several axes, and updates orthogonalised
by Newton-Schulz products.

A case is a dict of plain values; `kind` says which operator:

* ``attn_fwd``  `packed_attn_fwd` on the packed projection [T, (Hq + 2 Hkv) D]: every token sees its own sequence alone.
* ``attn_bwd``  `packed_attn_bwd`: the gradient of the projection from the output's.
* ``rope``      `rope_at_` in place on the query and key heads; with several axes each has its `sections` of the frequencies.
* ``orth``      `orthogonalize` on a list of matrices.
* ``muon``      one `muon_step` over a list of weight matrices.

The lengths of a case's sequences are dealt from its own values (`tokens`, `mean`, `deal`), so that its work is known; `tail` tokens at
the end belong to no sequence.  `shapes` lists matrices as "count x rows x columns".
"""
from __future__ import annotations

import math
import random

import torch

own = False

COEFFICIENTS = 3.4445, -4.7750, 2.0315      # of X, X X^T X and X X^T X X^T X
SCALE = 0.2                                 # an update's root mean square, times the learning rate


# ---------------------------------------------------------------------------------------------------------------- cases
def _attn(name, backward, tokens, q_heads, kv_heads, width, mean, deal, tail=0, causal=True, window=0):
    return _case(name=name, kind="attn_bwd" if backward else "attn_fwd", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads,
                 width=width, mean=mean, deal=deal, tail=tail, causal=causal, window=window)


def _rope(name, backward, tokens, heads, others, width, sections, table):
    return _case(name=name, kind="rope", backward=backward, tokens=tokens, heads=heads, others=others, width=width, sections=sections,
                 table=table)


def _orth(name, shapes, dtype):
    return _case(name=name, kind="orth", shapes=shapes, dtype=dtype)


def _muon(name, shapes, reduce, lr, decay, nesterov=True):
    return _case(name=name, kind="muon", shapes=shapes, reduce=reduce, lr=lr, decay=decay, nesterov=nesterov)


def _case(**values):
    return {k: v for k, v in values.items() if v is not None}


def listed():
    return [
        # a debugging job of the tiny decoder: a handful of sentences in 256 tokens
        _attn("packed_fwd_tiny", False, 256, 8, 8, 64, 40, 1),
        # a microbatch of a 1B model filled with documents of some hundred tokens, heads of 64 in groups of eight
        _attn("packed_fwd_1b", False, 8192, 32, 4, 64, 700, 2),
        # a long-context microbatch of a 7B model: a few documents of many thousand tokens, grouped heads of 128
        _attn("packed_fwd_long", False, 16384, 32, 8, 128, 9000, 3),
        # an encoder's batch of sentences, both directions, an odd number of tokens and a padded end
        _attn("packed_bwd_encoder", True, 2047, 12, 12, 64, 90, 4, tail=100, causal=False),
        # four sequences' worth of documents through a 7B block with grouped heads
        _attn("packed_bwd_7b", True, 16384, 32, 8, 128, 1500, 5),
        # the tiny decoder's heads by the positions within their documents
        _rope("rope_tiny", False, 255, 16, 8, 64, "32", 256),
        # time, height and width of image and video patches among text, gradient of a large microbatch
        _rope("rope_vision", True, 16384, 40, 8, 128, "16,24,24", 32768),
        # projections of a toy model: launches count
        _orth("orth_toy", "8x512x512,4x1376x512,4x512x1376", "bfloat16"),
        # sizes that are multiples of nothing
        _orth("orth_odd", "3x1000x333,1x4097x641,2x77x2050", "float32"),
        # every matrix of a model of two layers
        _muon("muon_toy", "8x128x128,2x512x128,2x128x512", "float32", 5e-5, 0.0, nesterov=False),
        # the matrices of 24 blocks of 1024, bf16 gradients
        _muon("muon_350m", "96x1024x1024,24x4096x1024,24x1024x4096", "bfloat16", 5e-5, 0.1),
        # a 7B block: four square projections, gate, up and down
        _muon("muon_7b", "4x4096x4096,2x11008x4096,1x4096x11008", "float32", 3e-5, 0.1),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["attn_fwd", "attn_bwd", "attn_fwd", "attn_bwd", "rope", "orth", "muon"])
    if kind.startswith("attn"):
        width = rng.choice([64, 128])
        kv = rng.choice([1, 2, 3, 4, 8])
        q = kv * rng.choice([1, 1, 2, 4, 5])
        tokens = log(2, 16384)
        causal = rng.random() < 0.8
        return _attn(None, kind == "attn_bwd", tokens, q, kv, width, log(1, 12000), rng.randrange(1 << 20),
                     rng.choice([0, 0, rng.randrange(tokens)]), causal, log(2, 4000) if causal and rng.random() < 0.25 else 0)
    if kind == "rope":
        width = rng.choice([32, 64, 96, 128, 256])
        axes = rng.choice([1, 1, 2, 3])
        cuts = sorted(rng.sample(range(1, width // 2), axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0, *cuts], [*cuts, width // 2]))
        heads, others = rng.randint(1, 40), rng.choice([0, 1, 4, 8])
        most = 16384 * 48 * 128 // ((heads + others) * width)
        return _rope(None, rng.random() < 0.5, log(1, min(30000, most)), heads, others, width, sections, log(16, 131072))
    shapes, left = [], 5e11
    for _ in range(rng.randint(1, 3)):
        rows, cols = log(8, 5000), log(8, 5000)
        n, m = min(rows, cols), max(rows, cols)
        count = min(rng.choice([1, 2, 5, 12]), int(left / (3 * n * n * m + n ** 3)), 60_000_000 // (rows * cols))
        if count > 0:
            left -= count * (3 * n * n * m + n ** 3)
            shapes.append(f"{count}x{rows}x{cols}")
    text = ",".join(shapes or ["1x64x96"])
    if kind == "orth":
        return _orth(None, text, rng.choice(["float32", "bfloat16"]))
    return _muon(None, text, rng.choice(["float32", "bfloat16"]), rng.uniform(1e-5, 7e-5), rng.choice([0.0, 0.1]), rng.random() < 0.7)


def _lengths(case):
    """Lengths of the sequences: spread about the mean as documents' are, an empty one here and there."""
    rng, left, out = random.Random(case["deal"]), case["tokens"] - case["tail"], []
    while left > 0:
        n = min(left, max(1, int(case["mean"] * math.exp(rng.gauss(-0.3, 0.8)))))
        out += [n, 0] if rng.random() < 0.02 else [n]
        left -= n
    return out


def _pairs(case):
    """How many keys are seen, summed over the tokens."""
    w, total = case["window"], 0
    for n in _lengths(case):
        if not case["causal"]:
            total += n * n
        elif 0 < w < n:
            total += w * (w + 1) // 2 + (n - w) * w
        else:
            total += n * (n + 1) // 2
    return total


def _shapes(text):
    return [tuple(int(x) for x in part.split("x")) for part in text.split(",")]


def _products(shapes):
    """Multiplications and additions of five iterations: both squares are symmetric, half of each is enough."""
    total = 0
    for count, rows, cols in shapes:
        n, m = min(rows, cols), max(rows, cols)
        total += count * 5 * (3 * n * n * m + n ** 3)
    return total


def work(case):
    c = case
    if c["kind"].startswith("attn"):
        T, Hq, d, qkv = c["tokens"], c["q_heads"], c["width"], (c["q_heads"] + 2 * c["kv_heads"]) * c["width"]
        if c["kind"] == "attn_fwd":
            return {"bytes": T * (2 * qkv + 2 * Hq * d + 4 * Hq), "flops": 4 * _pairs(c) * Hq * d}
        return {"bytes": T * (4 * qkv + 4 * Hq * d + 4 * Hq), "flops": 10 * _pairs(c) * Hq * d}
    if c["kind"] == "rope":
        T, n = c["tokens"], c["heads"] * c["width"]
        axes = c["sections"].count(",") + 1
        return {"bytes": T * (4 * n + 4 * axes) + 4 * min(T, c["table"]) * c["width"], "flops": 3 * T * n}
    shapes = _shapes(c["shapes"])
    n = sum(count * rows * cols for count, rows, cols in shapes)
    if c["kind"] == "orth":
        return {"bytes": n * ((4 if c["dtype"] == "float32" else 2) + 2), "flops": _products(shapes)}
    return {"bytes": n * (16 + 2 + (4 if c["reduce"] == "float32" else 2)), "flops": _products(shapes) + 8 * n}


# --------------------------------------------------------------------------------------------------------------- inputs
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def gradients(rows, cols, dtype):
        """Of a weight: a few directions stand out of noise whose size varies from row to row."""
        k = min(8, rows, cols)
        strong = normal(rows, k, dtype=torch.float32) @ normal(k, cols, dtype=torch.float32)
        return ((strong * 0.5 + normal(rows, cols, dtype=torch.float32)) * normal(rows, 1, dtype=torch.float32).exp() * 1e-3).to(dtype)

    st = {"case": dict(c)}
    if c["kind"].startswith("attn"):
        T, Hq, Hkv, d = c["tokens"], c["q_heads"], c["kv_heads"], c["width"]
        st["offsets"] = torch.tensor([0, *_lengths(c)], dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)
        st["qkv"] = normal(T, (Hq + 2 * Hkv) * d, scale=0.9)
        if c["kind"] == "attn_bwd":
            st["do"] = normal(T, Hq * d, scale=0.02)
            st["o"], st["lse"] = _plain_attn_fwd(st)
        if own:
            st["packed"] = _ops().pack_sequences(st["offsets"], T)     # made once for all layers of a batch
    elif c["kind"] == "rope":
        T, d, P = c["tokens"], c["width"], c["table"]
        st["sections"] = [int(x) for x in c["sections"].split(",")]
        inv = 500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d)
        a = torch.arange(P, dtype=torch.float64, device=dev)[:, None] * inv
        st["cs"] = torch.cat([a.cos(), a.sin()], 1).float()
        st["positions"] = torch.randint(0, P, (len(st["sections"]), T), generator=gen, device=dev, dtype=torch.int32)
        st["buf"] = normal(T, (c["heads"] + c["others"]) * d)
    elif c["kind"] == "orth":
        st["mats"] = [gradients(rows, cols, _DTYPES[c["dtype"]]) for count, rows, cols in _shapes(c["shapes"]) for _ in range(count)]
    else:
        sizes = [(rows, cols) for count, rows, cols in _shapes(c["shapes"]) for _ in range(count)]
        total = sum(r * k for r, k in sizes)
        flat = {"p": normal(total, scale=0.02, dtype=torch.float32), "p16": torch.zeros(total, dtype=torch.bfloat16, device=dev),
                "m": torch.empty(total, dtype=torch.float32, device=dev), "g": torch.empty(total, dtype=_DTYPES[c["reduce"]], device=dev)}
        views, at = {k: [] for k in flat}, 0
        for r, k in sizes:
            for name in flat:
                views[name].append(flat[name][at:at + r * k].view(r, k))
            views["g"][-1].copy_(gradients(r, k, torch.float32))
            views["m"][-1].copy_(gradients(r, k, torch.float32) * 4)
            at += r * k
        st |= {"flat": flat, "views": views, "hyper": {"lr": c["lr"], "momentum": 0.95, "weight_decay": c["decay"],
                                                       "nesterov": c["nesterov"], "grad_scale": 0.125}}
    return st


# ----------------------------------------------------------------------------------------------------------- plain forms
def _seen(st):
    """[T, T]: which keys (columns) a token (row) sees."""
    c, ends = st["case"], st["offsets"][1:].contiguous()
    t = torch.arange(c["tokens"], dtype=torch.int32, device=ends.device)
    doc = torch.searchsorted(ends, t, right=True)
    seen = (doc[:, None] == doc) & (doc < ends.numel())
    if c["causal"]:
        seen &= t[:, None] >= t
    if c["window"]:
        seen &= t[:, None] - t < c["window"]
    return seen


def _heads(st):
    """For each key head its query heads [rep, T, d], keys and values [T, d]."""
    c = st["case"]
    T, Hq, Hkv, d = c["tokens"], c["q_heads"], c["kv_heads"], c["width"]
    x = st["qkv"].view(T, Hq + 2 * Hkv, d).transpose(0, 1)
    rep = Hq // Hkv
    return [(slice(h * rep, (h + 1) * rep), x[h * rep:(h + 1) * rep].float(), x[Hq + h].float(), x[Hq + Hkv + h].float()) for h in range(Hkv)]


def _plain_attn_one(q, k, v, seen):
    s = (q @ k.t() / math.sqrt(q.shape[2])).masked_fill_(~seen, -math.inf)
    top = s.amax(2, keepdim=True)
    e = s.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = e.sum(2, keepdim=True)
    return e @ v / torch.where(total > 0, total, 1.0), (total.log() + top)[..., 0]


def _plain_attn_fwd(st):
    # one key head's group at a time: the scores of all heads at once are tens of gigabytes
    seen = _seen(st)
    parts = [_plain_attn_one(q, k, v, seen) for _, q, k, v in _heads(st)]
    o = torch.cat([o for o, _ in parts]).transpose(0, 1)
    return o.reshape(o.shape[0], -1).to(st["qkv"].dtype), torch.cat([lse for _, lse in parts])


def _plain_attn_bwd_one(q, k, v, do, o, lse, seen):
    scale = 1 / math.sqrt(q.shape[2])
    p = (q @ k.t()).mul_(scale).sub_(torch.where(lse > -math.inf, lse, 0.0)[..., None]).masked_fill_(~seen, -math.inf).exp_()
    dv = torch.einsum("htk,htd->kd", p, do)
    ds = (do @ v.t()).sub_((do * o).sum(2, keepdim=True)).mul_(p).mul_(scale)
    return ds @ k, torch.einsum("htk,htd->kd", ds, q), dv


def _plain_attn_bwd(st):
    c, seen = st["case"], _seen(st)
    T, Hq, d = c["tokens"], c["q_heads"], c["width"]
    do, o = (st[x].view(T, Hq, d).transpose(0, 1) for x in ("do", "o"))
    parts = [_plain_attn_bwd_one(q, k, v, do[h].float(), o[h].float(), st["lse"][h], seen) for h, q, k, v in _heads(st)]
    dq = torch.cat([p[0] for p in parts]).transpose(0, 1)
    dk, dv = (torch.stack([p[i] for p in parts], 1) for i in (1, 2))
    return torch.cat([dq, dk, dv], 1).reshape(T, -1).to(st["qkv"].dtype)


def _plain_rope(st):
    c, cs = st["case"], st["cs"]
    T, n, d, h = c["tokens"], c["heads"], c["width"], c["width"] // 2
    axis = torch.repeat_interleave(torch.arange(len(st["sections"]), device=cs.device), torch.tensor(st["sections"], device=cs.device))
    at = st["positions"].long()[axis].t()                              # [T, d / 2]: the position that turns each pair
    co, si = cs[:, :h].gather(0, at)[:, None], cs[:, h:].gather(0, at)[:, None]
    si = -si if c["backward"] else si
    x = st["buf"][:, :n * d].float().view(T, n, d)
    y = torch.cat([x[..., :h] * co - x[..., h:] * si, x[..., h:] * co + x[..., :h] * si], -1)
    st["buf"][:, :n * d] = y.view(T, n * d).to(st["buf"].dtype)
    return st["buf"]


def _plain_products(x, left):
    """One iteration after another, on the shorter side."""
    if left == 0:
        return x
    a, b, c = COEFFICIENTS
    s = x @ x.t()
    return _plain_products(a * x + (b * s + c * (s @ s)) @ x, left - 1)


def _plain_orth(u):
    norm = u.double().square().sum().sqrt().float()
    x = u.t() if u.shape[0] > u.shape[1] else u
    x = _plain_products(x / torch.where(norm > 0, norm, 1.0), 5)
    return x.t() if u.shape[0] > u.shape[1] else x


def _plain_muon_one(p, m, g, p16, h):
    g = g.float() * h["grad_scale"]
    m.copy_(m * h["momentum"] + g)
    o = _plain_orth(g + m * h["momentum"] if h["nesterov"] else m)
    p.copy_(p * (1 - h["lr"] * h["weight_decay"]) - h["lr"] * SCALE * math.sqrt(max(p.shape)) * o)
    p16.copy_(p)


def _plain_muon(st):
    v = st["views"]
    [_plain_muon_one(*each, st["hyper"]) for each in zip(v["p"], v["m"], v["g"], v["p16"])]
    return {k: st["flat"][k] for k in ("p", "p16", "m")}


# -------------------------------------------------------------------------------------------------------------------- run
def _ops():
    from zorse_b200.ops.api import get_ops

    return get_ops("sm100")


def run(state):
    if own:
        return _run_own(state)
    st, kind = state, state["case"]["kind"]
    if kind == "attn_fwd":
        return dict(zip(("out", "lse"), _plain_attn_fwd(st)))
    if kind == "attn_bwd":
        return _plain_attn_bwd(st)
    if kind == "rope":
        return _plain_rope(st)
    return [_plain_orth(x.float()).bfloat16() for x in st["mats"]] if kind == "orth" else _plain_muon(st)


def _run_own(st):
    ops, c = _ops(), st["case"]
    if c["kind"] == "attn_fwd":
        out, lse = ops.packed_attn_fwd(st["qkv"], st["packed"], c["q_heads"], c["kv_heads"], c["width"], c["causal"], c["window"])
        return {"out": out, "lse": lse}
    if c["kind"] == "attn_bwd":
        return ops.packed_attn_bwd(st["do"], st["qkv"], st["o"], st["lse"], st["packed"], c["q_heads"], c["kv_heads"], c["width"],
                                   c["causal"], c["window"])
    if c["kind"] == "rope":
        return ops.rope_at_(st["buf"], st["cs"], st["positions"], c["heads"], c["width"], st["sections"], backward=c["backward"])
    if c["kind"] == "orth":
        return ops.orthogonalize(st["mats"])
    v = st["views"]
    ops.muon_step(v["p"], v["m"], v["g"], v["p16"], **st["hyper"])
    return {k: st["flat"][k] for k in ("p", "p16", "m")}


# ---------------------------------------------------------------------------------------------------------- 64-bit answers
def _exact_orth(u):
    """The polynomials applied to the singular values through the Gram matrix of the shorter side, which they commute with."""
    wide = u.shape[0] <= u.shape[1]
    a, b, c = COEFFICIENTS
    norm2 = (u * u).sum()
    gram = (u @ u.t() if wide else u.t() @ u) / torch.where(norm2 > 0, norm2, 1.0)
    whole = torch.eye(gram.shape[0], dtype=u.dtype, device=u.device)
    for _ in range(5):     # X -> q(G) X, so G = X X^T -> q(G) G q(G), and the factors multiply up
        q = c * (gram @ gram) + b * gram
        q.diagonal().add_(a)
        whole, gram = q @ whole, q @ gram @ q
    x = u / torch.where(norm2 > 0, norm2.sqrt(), 1.0)
    return whole @ x if wide else x @ whole


def _exact_attn(st):
    c = st["case"]
    T, Hq, Hkv, d, w = c["tokens"], c["q_heads"], c["kv_heads"], c["width"], c["window"]
    rep, scale, dev = Hq // Hkv, d ** -0.5, st["qkv"].device
    back = c["kind"] == "attn_bwd"
    x = st["qkv"].view(T, Hq + 2 * Hkv, d)
    out = torch.zeros(T, Hq + 2 * Hkv if back else Hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((Hq, T), -math.inf, dtype=torch.float64, device=dev)
    bounds = [0]
    for n in _lengths(c):
        bounds.append(bounds[-1] + n)
    for lo, hi in zip(bounds, bounds[1:]):
        n = hi - lo
        if n == 0:
            continue
        hide = None
        if c["causal"]:
            ones = torch.ones(n, n, dtype=torch.bool, device=dev)
            hide = ones.triu(1) | ones.tril(-w) if w else ones.triu(1)
        step = Hkv if n <= 1024 else 1
        for k0 in range(0, Hkv, step):
            q = x[lo:hi, k0 * rep:(k0 + step) * rep].double().view(n, step, rep, d)
            k = x[lo:hi, Hq + k0:Hq + k0 + step].double()
            v = x[lo:hi, Hq + Hkv + k0:Hq + Hkv + k0 + step].double()
            if n > 1024:     # query heads one by one: a long sequence's scores in 64 bits are gigabytes
                groups = [(r, r + 1) for r in range(rep)]
            else:
                groups = [(0, rep)]
            for r0, r1 in groups:
                qq = q[:, :, r0:r1]
                s = torch.einsum("qgrd,kgd->grqk", qq, k) * scale
                if hide is not None:
                    s.masked_fill_(hide, -math.inf)
                hs = [(k0 + i) * rep + r for i in range(step) for r in range(r0, r1)]
                if not back:
                    total = torch.logsumexp(s, 3)
                    lse[hs, lo:hi] = total.view(-1, n)
                    o = torch.einsum("grqk,kgd->qgrd", (s - total[..., None]).exp_(), v)
                    out[lo:hi, hs] = o.reshape(n, -1, d)
                    continue
                g = st["do"].view(T, Hq, d)[lo:hi, hs].double().view(n, step, r1 - r0, d)
                dot = (g * st["o"].view(T, Hq, d)[lo:hi, hs].double().view(n, step, r1 - r0, d)).sum(3)
                p = s.sub_(st["lse"][hs, lo:hi].double().view(step, r1 - r0, n, 1)).exp_()
                out[lo:hi, Hq + Hkv + k0:Hq + Hkv + k0 + step] += torch.einsum("grqk,qgrd->kgd", p, g)
                p *= torch.einsum("qgrd,kgd->grqk", g, v) - dot.permute(1, 2, 0)[..., None]
                out[lo:hi, hs] = (torch.einsum("grqk,kgd->qgrd", p, k) * scale).reshape(n, -1, d)
                out[lo:hi, Hq + k0:Hq + k0 + step] += torch.einsum("grqk,qgrd->kgd", p, qq) * scale
    return out.view(T, -1) if back else {"out": out.view(T, -1), "lse": lse}


def exact(case, seed):
    """What `run` returns for the inputs of this seed, in 64 bits."""
    st, c = prepare(case, seed), case
    if c["kind"].startswith("attn"):
        return _exact_attn(st)
    if c["kind"] == "rope":
        T, n, d, h = c["tokens"], c["heads"], c["width"], c["width"] // 2
        z, at = st["buf"].double(), 0
        x = z[:, :n * d].reshape(T, n, 2, h)
        x = torch.complex(x[:, :, 0].contiguous(), x[:, :, 1].contiguous())
        for axis, size in enumerate(st["sections"]):
            rows = st["cs"][st["positions"][axis].long()].double()
            turn = torch.complex(rows[:, at:at + size].contiguous(), rows[:, h + at:h + at + size].contiguous())
            x[:, :, at:at + size] *= (turn.conj() if c["backward"] else turn)[:, None]
            at += size
        z[:, :n * d] = torch.cat([x.real, x.imag], -1).view(T, n * d)
        return z
    if c["kind"] == "orth":
        return [_exact_orth(x.double()) for x in st["mats"]]
    h, f = st["hyper"], st["flat"]
    out = {k: f[k].double() for k in ("p", "p16", "m")}
    at = 0
    for g in st["views"]["g"]:
        p, p16, m = (out[k][at:at + g.numel()].view(g.shape) for k in ("p", "p16", "m"))
        at += g.numel()
        g = g.double() * h["grad_scale"]
        m.mul_(h["momentum"]).add_(g)
        o = _exact_orth(g + h["momentum"] * m if h["nesterov"] else m)
        p -= h["lr"] * (h["weight_decay"] * p + SCALE * max(p.shape) ** 0.5 * o)
        p16.copy_(p)
    return out
