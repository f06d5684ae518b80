"""The measured calls of three operators of a distillation step, in their plain form and as the framework runs them.

``qk``     norm of each query and key head and the rotation of its position, forward and backward
           (``voodoo_quant.fused_blocks.qk_norm_rope``);
``embed``  lookup of token rows in a gated embedding (the softmax mixture of packed GGUF candidates), scaled, and
           the gradient of the mixture's probabilities, summed over the sorted tokens
           (``voodoo_quant.layers.gated_embedding``);
``clip``   the global norm of many gradients and their clipping in place
           (``voodoo_quant.training.grad_clip.clip_grad_norm_``).

``own`` chooses between the two forms.  The plain forms compute in 32 bits (sums of many terms in 64) and round once.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

BF16, F16, F32 = "bfloat16", "float16", "float32"
EPS = 1e-6

# bytes of one block and the weights it holds, by format
BLOCK_BYTES = {"Q8_0": 34, "Q2_K": 84, "Q3_K": 110, "Q4_K": 144, "Q5_K": 176, "Q6_K": 210, "IQ4_XS": 136}
BLOCK_ELEMS = {"Q8_0": 32}
ALL_K = "Q2_K,Q3_K,Q4_K,Q5_K,Q6_K,Q8_0"
K7 = "IQ4_XS,Q3_K,Q4_K,Q5_K,Q6_K,Q8_0,Q2_K"
# byte offsets of the 16-bit scales inside a block
SCALE_AT = {"Q8_0": (0,), "Q2_K": (80, 82), "Q3_K": (108,), "Q4_K": (0, 2), "Q5_K": (0, 2), "Q6_K": (208,),
            "IQ4_XS": (0,)}
# a scale that gives weights of about 0.02
SCALE_OF = {"Q8_0": 2.0 ** -12, "Q2_K": 2.0 ** -9, "Q3_K": 2.0 ** -11, "Q4_K": 2.0 ** -13, "Q5_K": 2.0 ** -14,
            "Q6_K": 2.0 ** -15, "IQ4_XS": 2.0 ** -16}
IQ4 = (-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113)


# ------------------------------------------------------------------ cases
def _qk(name, batch, seq, heads, kv_heads, dim, rotary, dtype, fused, grad, offset=0.0, first=0):
    c = {"op": "qk", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
         "dtype": dtype, "fused": fused, "grad": grad, "offset": offset, "first": first}
    return dict(c, name=name) if name else c


def _embed(name, tokens, vocab, dim, types, zipf, scale, grad, start=0, rows=None):
    c = {"op": "embed", "tokens": tokens, "vocab": vocab, "dim": dim, "types": types, "zipf": zipf, "scale": scale,
         "grad": grad, "start": start, "rows": vocab if rows is None else rows}
    return dict(c, name=name) if name else c


def _clip(name, kind, tensors, size, dtype, max_norm):
    c = {"op": "clip", "kind": kind, "tensors": tensors, "size": size, "dtype": dtype, "max_norm": max_norm}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of the 0.6B decoder's head layout, as a generating model calls it
        _qk("qk one token", 1, 1, 16, 8, 128, 128, BF16, True, False, first=70001),
        # a short float32 batch of the tiny configuration, with its gradients
        _qk("qk tiny float32", 2, 127, 4, 4, 64, 64, F32, False, True),
        # odd lengths, a head of 96 of which 32 values turn, weights stored as their distance from one
        _qk("qk ragged float16", 3, 1021, 14, 2, 96, 32, F16, True, True, offset=1.0),
        # the 0.6B decoder's training batch
        _qk("qk train 0.6b", 8, 2048, 16, 8, 128, 128, BF16, True, True),
        # the 8B decoder's training batch
        _qk("qk train 8b", 4, 4096, 32, 8, 128, 128, BF16, True, True),
        # a few tokens of the 8B table, forward only: a teacher or a generating model
        _embed("embed few tokens", 5, 128256, 4096, ALL_K, False, 1.0, False),
        # odd sizes: 1000 of 1024 stored columns, scaled rows
        _embed("embed ragged", 777, 5003, 1000, "Q4_K,IQ4_XS,Q8_0", True, math.sqrt(1000.0), True),
        # the 8B training batch over text, where few words make most of the tokens
        _embed("embed train 8b text", 16384, 128256, 4096, ALL_K, True, 1.0, True),
        # one of four vocabulary shards of the 32B decoder, uniform tokens
        _embed("embed train 32b shard", 16384, 152064, 5120, K7, False, 1.0, True, start=38016, rows=38016),
        # the gates of the 8B decoder: 226 tensors of six values
        _clip("clip gates 8b", "even", 226, 6, F32, 1.0),
        # gradients of low-rank factors beside float32 gates, odd sizes
        _clip("clip adapters", "ragged", 150, 40961, "mixed", 0.5),
        # every gradient of a dense 0.6B decoder
        _clip("clip dense 0.6b", "decoder", 28, 1024, BF16, 1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["qk", "embed", "clip"])
    if op == "qk":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        rotary = rng.choice([dim, dim, dim // 32 * 16])
        batch, kv = rng.randint(1, 8), rng.choice([1, 2, 4, 8])
        heads = kv * rng.randint(1, 5)
        most = 4 * 4096 * 40 * 128 // (batch * (heads + kv) * dim)
        dtype = rng.choice([BF16, BF16, F16, F32])
        if dtype == F32:
            most //= 2
        return _qk("", batch, _log(rng, 1, max(2, min(most, 16384))), heads, kv, dim, rotary, dtype,
                   rng.random() < 0.5, rng.random() < 0.7, rng.choice([0.0, 0.0, 1.0]), rng.randint(0, 100000))
    if op == "embed":
        types = rng.sample(sorted(BLOCK_BYTES), rng.randint(1, 7))
        dim = 8 * _log(rng, 32, 640)
        vocab = _log(rng, 1000, 130000)
        rows = vocab if rng.random() < 0.6 else vocab // 2 + 1
        return _embed("", _log(rng, 1, 16384), vocab, dim, ",".join(types), rng.random() < 0.6,
                      rng.choice([1.0, math.sqrt(dim)]), rng.random() < 0.8, rng.randint(0, vocab - rows), rows)
    return _clip("", rng.choice(["even", "ragged"]), rng.randint(2, 500), _log(rng, 1, 200000),
                 rng.choice([F32, BF16, F16, "mixed"]), rng.choice([0.1, 1.0, 1e9]))


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _prepare_qk(c, g):
    dt = getattr(torch, c["dtype"])
    b, s, hq, hk, d, r = (c[k] for k in ("batch", "seq", "heads", "kv_heads", "dim", "rotary"))
    if c["fused"]:  # column ranges of one projection's output
        qkv = _normal((b, s, (hq + 2 * hk) * d), g, dt)
        q, k, _ = qkv.split([hq * d, hk * d, hk * d], dim=-1)
        q, k = q.view(b, s, hq, d), k.view(b, s, hk, d)
    else:
        q, k = _normal((b, s, hq, d), g, dt), _normal((b, s, hk, d), g, dt)
    st = {"op": "qk", "q": q, "k": k, "eps": EPS, "offset": c["offset"], "grad": c["grad"]}
    st["wq"] = (1.0 - c["offset"] + _normal((d,), g, scale=0.1)).to(dt)
    st["wk"] = (1.0 - c["offset"] + _normal((d,), g, scale=0.1)).to(dt)
    pos = torch.arange(c["first"], c["first"] + s, device="cuda", dtype=torch.float64)
    angle = pos[:, None] * (1e4 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r))
    angle = torch.cat([angle, angle], dim=-1)[None]
    st["cos"], st["sin"] = angle.cos().to(dt), angle.sin().to(dt)
    if c["grad"]:
        st["gq"], st["gk"] = _normal((b, s, hq, d), g, dt), _normal((b, s, hk, d), g, dt)
        st["leaves"] = [t.requires_grad_(True) for t in (q.detach(), k.detach(), st["wq"], st["wk"])]
        st["q"], st["k"] = st["leaves"][:2]
    return st


def _blocks(fmt, rows, cols, g):
    """Packed blocks [rows, blocks * bytes] of a table: random codes and small scales, a few percent apart."""
    nb, bb = cols // BLOCK_ELEMS.get(fmt, 256), BLOCK_BYTES[fmt]
    q = torch.randint(0, 256, (rows * nb, bb), generator=g, device="cuda", dtype=torch.uint8)
    for at in SCALE_AT[fmt]:
        d = (torch.rand(rows * nb, 1, generator=g, device="cuda") + 0.5) * SCALE_OF[fmt]
        q[:, at:at + 2] = d.to(torch.float16).view(torch.uint8)
    return q


def _zipf(vocab):
    """Probability of the i-th most frequent of `vocab` words."""
    p = 1.0 / torch.arange(1, vocab + 1, dtype=torch.float64)
    return p / p.sum()


def _prepare_embed(c, g):
    v, d, t, rows = c["vocab"], c["dim"], c["tokens"], c["rows"]
    types = c["types"].split(",")
    padded = (d + 255) // 256 * 256
    if c["zipf"]:
        rank = torch.searchsorted(_zipf(v).cumsum(0).cuda(),
                                  torch.rand(t, generator=g, device="cuda", dtype=torch.float64)).clamp_(max=v - 1)
        ids = torch.randperm(v, generator=g, device="cuda")[rank]
    else:
        ids = torch.randint(0, v, (t,), generator=g, device="cuda")
    probs = torch.softmax(_normal((len(types),), g), 0)
    st = {"op": "embed", "types": types, "blocks": [_blocks(f, rows, padded, g) for f in types], "ids": ids,
          "probs": probs.requires_grad_(c["grad"]), "rows": rows, "dim": d, "padded": padded, "start": c["start"],
          "scale": c["scale"], "grad": c["grad"]}
    if c["grad"]:
        st["dy"] = _normal((t, d), g, torch.bfloat16, 1e-3)
    return st


def _clip_shapes(c):
    """(shape, dtype name) of each gradient."""
    n, size = c["tensors"], c["size"]
    if c["kind"] == "decoder":  # `n` layers of hidden width `size`: attention, MLP, norms; the tied embedding
        kv, ffn = size, 3 * size - 64
        layer = [(2 * size, size), (kv, size), (kv, size), (size, 2 * size), (ffn, size), (ffn, size), (size, ffn),
                 (size,), (size,), (128,), (128,)]
        return [(s, c["dtype"]) for s in [(151936, size)] + layer * n + [(size,)]]
    sizes = [size] * n if c["kind"] == "even" else [1 + (7919 * i * i + 31 * i) % size for i in range(n)]
    kinds = [F32, BF16] if c["dtype"] == "mixed" else [c["dtype"]]
    return [((s,), kinds[i % len(kinds)]) for i, s in enumerate(sizes)]


def _prepare_clip(c, g):
    shapes = _clip_shapes(c)
    flat, params = {}, [None] * len(shapes)
    for kind in sorted({k for _, k in shapes}):
        sizes = [math.prod(s) for s, k in shapes if k == kind]
        dt = getattr(torch, kind)
        flat[kind] = torch.empty(sum(sizes), device="cuda", dtype=dt).normal_(0.0, 0.1, generator=g)
        parts = iter(flat[kind].split(sizes))
        for i, (s, k) in enumerate(shapes):
            if k == kind:
                params[i] = torch.zeros(s, device="cuda", dtype=dt, requires_grad=True)
                params[i].grad = next(parts).view(s)
    return {"op": "clip", "flat": flat, "params": params, "max_norm": c["max_norm"]}


def prepare(case, seed):
    g = _generator(seed)
    return {"qk": _prepare_qk, "embed": _prepare_embed, "clip": _prepare_clip}[case["op"]](case, g)


# ------------------------------------------------------------------ plain forms
def _norm_rope(x, w, cos, sin, eps, offset):
    """The turned heads, and what their gradient needs."""
    xf, wf = x.float(), w.float() + offset
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps)
    n = xf * r
    y = n * wf
    c, s = cos.float().unsqueeze(2), sin.float().unsqueeze(2)
    rot, h = c.shape[-1], c.shape[-1] // 2
    a, b = y[..., :h], y[..., h:rot]
    out = torch.cat([a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:], y[..., rot:]], dim=-1)
    return out.to(x.dtype), (n, r, wf, c, s)


def _norm_rope_gradient(g, x, w, saved):
    n, r, wf, c, s = saved
    rot, h = c.shape[-1], c.shape[-1] // 2
    gf = g.float()
    a, b = gf[..., :h], gf[..., h:rot]
    gy = torch.cat([a * c[..., :h] + b * s[..., h:], b * c[..., h:] - a * s[..., :h], gf[..., rot:]], dim=-1)
    dw = (gy * n).sum((0, 1, 2), dtype=torch.float64)
    gn = gy * wf
    dx = r * (gn - n * (gn * n).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw.to(w.dtype)


def _plain_qk(st):
    with torch.no_grad():
        q, sq = _norm_rope(st["q"], st["wq"], st["cos"], st["sin"], st["eps"], st["offset"])
        k, sk = _norm_rope(st["k"], st["wk"], st["cos"], st["sin"], st["eps"], st["offset"])
        if not st["grad"]:
            return q, k
        dq, dwq = _norm_rope_gradient(st["gq"], st["q"], st["wq"], sq)
        dk, dwk = _norm_rope_gradient(st["gk"], st["k"], st["wk"], sk)
    return q, k, dq, dk, dwq, dwk


def _half(b):
    return b.contiguous().view(torch.float16).float()


def _six_bit(q):
    """Scales and minima [.., 8] of the 12-byte tables of Q4_K and Q5_K."""
    lo, mid, hi = q[:, 0:4], q[:, 4:8], q[:, 8:12]
    sc = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], dim=1)
    mn = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], dim=1)
    return sc.float(), mn.float()


def _nibbles(q):
    """[n, 128] bytes of four 64-weight groups -> [n, 8, 32]: low nibbles, then high ones."""
    q = q.view(-1, 4, 1, 32)
    return torch.cat([q & 15, q >> 4], dim=2).reshape(-1, 8, 32)


def _pairs(q):
    """[n, 64] bytes -> [n, 2, 4, 32]: two bits of each byte at a time."""
    q = q.view(-1, 2, 1, 32)
    return torch.cat([(q >> (2 * i)) & 3 for i in range(4)], dim=2)


def _decode(fmt, b):
    """float32 weights [n, 256] (Q8_0: [n, 32]) of packed blocks [n, bytes]."""
    if fmt == "Q8_0":
        return _half(b[:, :2]) * b[:, 2:].contiguous().view(torch.int8).float()
    if fmt == "Q4_K":
        sc, mn = _six_bit(b[:, 4:16])
        q = _nibbles(b[:, 16:144]).float()
        return ((_half(b[:, 0:2]) * sc).unsqueeze(2) * q - (_half(b[:, 2:4]) * mn).unsqueeze(2)).view(-1, 256)
    if fmt == "Q5_K":
        sc, mn = _six_bit(b[:, 4:16])
        high = torch.stack([(b[:, 16:48] >> i) & 1 for i in range(8)], dim=1)
        q = (_nibbles(b[:, 48:176]) | (high << 4)).float()
        return ((_half(b[:, 0:2]) * sc).unsqueeze(2) * q - (_half(b[:, 2:4]) * mn).unsqueeze(2)).view(-1, 256)
    if fmt == "Q6_K":
        low = b[:, :128].view(-1, 2, 1, 64)
        low = torch.cat([low & 15, low >> 4], dim=2).view(-1, 2, 4, 32)
        q = (low | (_pairs(b[:, 128:192]) << 4)).float() - 32.0
        sc = _half(b[:, 208:210]) * b[:, 192:208].contiguous().view(torch.int8).float()
        return (sc.unsqueeze(2) * q.view(-1, 16, 16)).view(-1, 256)
    if fmt == "Q2_K":
        sc = _half(b[:, 80:82]) * (b[:, :16] & 15).float()
        mn = _half(b[:, 82:84]) * (b[:, :16] >> 4).float()
        return (sc.unsqueeze(2) * _pairs(b[:, 16:80]).float().view(-1, 16, 16) - mn.unsqueeze(2)).view(-1, 256)
    if fmt == "Q3_K":
        high = torch.stack([(b[:, :32] >> i) & 1 for i in range(8)], dim=1).view(-1, 2, 4, 32)
        q = (_pairs(b[:, 32:96]) | (high << 2)).float() - 4.0
        t = b[:, 96:108]
        low = torch.cat([t[:, :8] & 15, t[:, :8] >> 4], dim=1)
        top = torch.cat([(t[:, 8:] >> (2 * i)) & 3 for i in range(4)], dim=1)
        sc = _half(b[:, 108:110]) * ((low | (top << 4)).float() - 32.0)
        return (sc.unsqueeze(2) * q.view(-1, 16, 16)).view(-1, 256)
    if fmt == "IQ4_XS":
        top = b[:, 2:4].contiguous().view(torch.int16).int() & 0xFFFF
        top = torch.cat([(top >> (2 * i)) & 3 for i in range(8)], dim=1)
        low = torch.stack([b[:, 4:8] & 15, b[:, 4:8] >> 4], dim=2).view(-1, 8).int()
        sc = _half(b[:, 0:2]) * ((low | (top << 4)).float() - 32.0)
        q = b[:, 8:136].view(-1, 8, 1, 16)
        q = torch.cat([q & 15, q >> 4], dim=2).view(-1, 8, 32)
        return (sc.unsqueeze(2) * torch.tensor(IQ4, device=b.device, dtype=torch.float32)[q.long()]).view(-1, 256)
    raise ValueError(fmt)


def _plain_embed(st):
    with torch.no_grad():
        local = st["ids"] - st["start"]
        here = (local >= 0) & (local < st["rows"])
        local = local.clamp(0, st["rows"] - 1)
        d, t = st["dim"], local.numel()
        mixed, grads = torch.zeros(t, d, device="cuda"), []
        dy = st["dy"].float() * (here.float() * st["scale"]).unsqueeze(1) if st["grad"] else None
        for k, (fmt, q) in enumerate(zip(st["types"], st["blocks"])):
            b = q.view(st["rows"], -1).index_select(0, local).view(-1, BLOCK_BYTES[fmt])
            w = _decode(fmt, b).view(t, st["padded"])[:, :d]
            mixed += st["probs"][k] * w
            if st["grad"]:
                grads.append((dy * w).sum(dtype=torch.float64))
        out = (mixed * (here.float() * st["scale"]).unsqueeze(1)).to(torch.bfloat16)
        return (out, torch.stack(grads).float()) if st["grad"] else out


def _plain_clip(st):
    grads = [p.grad for p in st["params"]]
    flat = torch.cat([g.reshape(-1).float() for g in grads])
    norm = flat.double().square().sum().sqrt().float()
    flat *= torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    torch._foreach_copy_([g.view(-1) for g in grads], list(flat.split([g.numel() for g in grads])))
    return norm, st["flat"]


# ------------------------------------------------------------------ the framework's calls
def _package():
    if "voodoo_quant" in sys.modules:
        return
    p = str(Path("voodoo-dyn-quant_b200").resolve())
    if p not in sys.path:
        sys.path.insert(0, p)


def _own_qk(st):
    from voodoo_quant.fused_blocks import qk_norm_rope

    if not st["grad"]:
        with torch.no_grad():
            return qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], st["eps"],
                                weight_offset=st["offset"])
    q, k = qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], st["eps"],
                        weight_offset=st["offset"])
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), st["leaves"], (st["gq"], st["gk"])))


def _own_embed(st):
    from voodoo_quant.layers import gated_embedding

    out = gated_embedding(st["ids"], st["probs"], st["types"], st["blocks"], st["rows"], st["dim"], scale=st["scale"],
                          vocab_start=st["start"])
    if not st["grad"]:
        return out
    return out.detach(), torch.autograd.grad(out, st["probs"], st["dy"])[0]


def _own_clip(st):
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    return clip_grad_norm_(st["params"], st["max_norm"]), st["flat"]


def run(state):
    if own:
        _package()
        return {"qk": _own_qk, "embed": _own_embed, "clip": _own_clip}[state["op"]](state)
    return {"qk": _plain_qk, "embed": _plain_embed, "clip": _plain_clip}[state["op"]](state)


# ------------------------------------------------------------------ the work of one pass
def _row_bytes(c):
    padded = (c["dim"] + 255) // 256 * 256
    return sum(padded // BLOCK_ELEMS.get(f, 256) * BLOCK_BYTES[f] for f in c["types"].split(","))


def _distinct(c):
    """Expected distinct rows of this shard that the tokens name."""
    p = _zipf(c["vocab"]).numpy() if c["zipf"] else np.full(c["vocab"], 1.0 / c["vocab"])
    return float(-np.expm1(c["tokens"] * np.log1p(-p)).sum()) * c["rows"] / c["vocab"]


def work(case):
    c = case
    if c["op"] == "qk":
        size = 4 if c["dtype"] == F32 else 2
        n = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        small = 2 * c["seq"] * c["rotary"] * size + 2 * c["dim"] * size * (2 if c["grad"] else 1)
        return {"bytes": n * size * (4 if c["grad"] else 2) + small, "flops": n * (22 if c["grad"] else 8)}
    if c["op"] == "embed":
        k, u = len(c["types"].split(",")), _distinct(c)
        n = c["tokens"] * c["dim"]
        read = u * _row_bytes(c) + c["tokens"] * 8 + 4 * k
        if not c["grad"]:
            return {"bytes": read + 2 * n, "flops": u * c["dim"] * 4 * k}
        return {"bytes": read + 4 * n + 4 * k, "flops": u * c["dim"] * 6 * k + n}
    n = sum(math.prod(s) * (4 if k == F32 else 2) for s, k in _clip_shapes(c))
    return {"bytes": 2 * n, "flops": 3 * sum(math.prod(s) for s, _ in _clip_shapes(c))}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_heads(x, w, cos, sin, eps, offset):
    """Heads over their root mean square, weighted; the first places then turned in pairs (j, j + h), h half of them."""
    y = x / torch.sqrt(torch.mean(x.square(), dim=-1, keepdim=True) + eps) * (w + offset)
    rot = cos.shape[-1]
    turned = y[..., :rot]
    partner = torch.roll(turned, rot // 2, dims=-1)
    sign = torch.ones(rot, device=x.device, dtype=torch.float64)
    sign[: rot // 2] = -1.0
    turned = turned * cos[:, :, None] + partner * sign * sin[:, :, None]
    return torch.cat([turned, y[..., rot:]], dim=-1)


def _exact_qk(case, st):
    x = [t.detach().double().requires_grad_(case["grad"]) for t in (st["q"], st["k"], st["wq"], st["wk"])]
    cos, sin = st["cos"].double(), st["sin"].double()
    q = _exact_heads(x[0], x[2], cos, sin, st["eps"], st["offset"])
    k = _exact_heads(x[1], x[3], cos, sin, st["eps"], st["offset"])
    if not case["grad"]:
        return q, k
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), x, (st["gq"].double(), st["gk"].double())))


def _exact_fields(fmt):
    """Of each of the 256 (Q8_0: 32) weights: its scale's number and the bit fields (byte, shift, bits, place in the
    code) of its code."""
    if fmt == "Q8_0":
        e = np.arange(32)
        return e * 0, [(2 + e, e * 0, 8, 0)]
    e = np.arange(256)
    half, l128, l32 = e // 128, e % 128, e % 32
    if fmt in ("Q4_K", "Q5_K"):
        at = 16 if fmt == "Q4_K" else 48
        f = [(at + e // 64 * 32 + l32, e // 32 % 2 * 4, 4, 0)]
        if fmt == "Q5_K":
            f.append((16 + l32, e // 32, 1, 4))
        return e // 32, f
    if fmt == "Q6_K":
        return e // 16, [(64 * half + l128 % 64, l128 // 64 * 4, 4, 0), (128 + 32 * half + l32, l128 // 32 * 2, 2, 4)]
    if fmt == "Q2_K":
        return e // 16, [(16 + 32 * half + l32, l128 // 32 * 2, 2, 0)]
    if fmt == "Q3_K":
        return e // 16, [(32 + 32 * half + l32, l128 // 32 * 2, 2, 0), (l32, e // 32, 1, 2)]
    return e // 32, [(8 + e // 32 * 16 + e % 16, e % 32 // 16 * 4, 4, 0)]  # IQ4_XS


def _exact_scales(fmt, b):
    """(scale, minimum) [n, scales] in 64 bits of blocks [n, bytes] held as int64."""
    def half(at):
        bits = (b[:, at] | (b[:, at + 1] << 8)).to(torch.int32).to(torch.int16)
        return bits.view(torch.float16).double()[:, None]

    def signed(t):
        return torch.where(t > 127, t - 256, t).double()

    def columns(f, n):
        return torch.stack([f(j) for j in range(n)], dim=1)

    if fmt == "Q8_0":
        return half(0), None
    if fmt in ("Q4_K", "Q5_K"):
        sc = columns(lambda j: b[:, 4 + j] % 64 if j < 4 else b[:, 8 + j] % 16 + b[:, j] // 64 * 16, 8)
        mn = columns(lambda j: b[:, 8 + j] % 64 if j < 4 else b[:, 8 + j] // 16 + b[:, 4 + j] // 64 * 16, 8)
        return half(0) * sc.double(), half(2) * mn.double()
    if fmt == "Q6_K":
        return half(208) * signed(b[:, 192:208]), None
    if fmt == "Q2_K":
        return half(80) * (b[:, :16] % 16).double(), half(82) * (b[:, :16] // 16).double()
    if fmt == "Q3_K":
        sc = columns(lambda j: (b[:, 96 + j % 8] >> (j // 8 * 4)) % 16 + (b[:, 104 + j % 4] >> (j // 4 * 2)) % 4 * 16, 16)
        return half(108) * (sc - 32).double(), None
    sc = columns(lambda j: (b[:, 4 + j // 2] >> (j % 2 * 4)) % 16 + (b[:, 2 + j // 4] >> (j % 4 * 2)) % 4 * 16, 8)
    return half(0) * (sc - 32).double(), None


def _exact_weights(fmt, b):
    """Weights [n, 256 or 32] in 64 bits of packed blocks [n, bytes]."""
    b = b.long()
    which, fields = _exact_fields(fmt)

    def dev(a):
        return torch.as_tensor(np.ascontiguousarray(a), device=b.device)

    code = sum(((b[:, dev(at)] >> dev(shift)) % 2 ** bits) << place for at, shift, bits, place in fields)
    if fmt == "Q8_0":
        code = torch.where(code > 127, code - 256, code)
    elif fmt == "IQ4_XS":
        code = torch.tensor(IQ4, device=b.device)[code]
    code = code - {"Q6_K": 32, "Q3_K": 4}.get(fmt, 0)
    scale, low = _exact_scales(fmt, b)
    w = scale[:, dev(which)] * code.double()
    return w if low is None else w - low[:, dev(which)]


def _exact_embed(case, st):
    p = st["probs"].detach().double()
    out = torch.zeros(case["tokens"], case["dim"], device="cuda", dtype=torch.float64)
    grad = torch.zeros(len(st["types"]), device="cuda", dtype=torch.float64)
    mine = ((st["ids"] >= case["start"]) & (st["ids"] < case["start"] + case["rows"])).nonzero()[:, 0]
    for part in mine.split(1024):
        rows = st["ids"][part] - case["start"]
        for k, fmt in enumerate(st["types"]):
            b = st["blocks"][k].view(case["rows"], -1)[rows].view(-1, BLOCK_BYTES[fmt])
            w = _exact_weights(fmt, b).view(len(part), -1)[:, : case["dim"]] * case["scale"]
            out[part] += p[k] * w
            if case["grad"]:
                grad[k] += (w * st["dy"][part].double()).sum()
    return (out, grad) if case["grad"] else out


def _exact_clip(case, st):
    norm = torch.sqrt(sum(torch.linalg.vector_norm(f.double()).square() for f in st["flat"].values()))
    scale = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    return norm, {k: f.double() * scale for k, f in st["flat"].items()}


def exact(case, seed):
    st = prepare(case, seed)
    return {"qk": _exact_qk, "embed": _exact_embed, "clip": _exact_clip}[case["op"]](case, st)
