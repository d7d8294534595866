"""The parts of a mixture-of-experts layer around its quantized products, and the
layer for a few tokens: what is measured, and what it is compared with.

Three operators of `Context`:

  rms_norm    the residual's addition, the RMS norm and the norm's output in
              8-bit blocks (Q8_K or Q8_0), the right-hand side that the quantized
              products take
  moe_route   the router's product with its f32 weights, the softmax or sigmoid,
              and the best experts of each token with their weights
  moe_ffn     the chosen experts' gate, up and down products, SiLU between them and
              the weighted sum over a token's experts

`run` computes them in torch's elementary operations, or, where `own` is set, by
the framework's calls.

The norm is the reference's sequence of f32 operations (the squares summed in 64
bits), so that its 8-bit levels are defined to the last one.  Router and layer keep
their sums in 64 bits and round once where a number becomes an f32: the logits, a
token's weights, the gate and up products, their SiLU product, the result.  The
products see their activations in 8-bit blocks.
"""
import importlib

import torch

own = False  # True: `run` makes the framework's calls

F32, F64, I32 = torch.float32, torch.float64, torch.int32
BLOCK = {"Q8_0": 32, "Q2_K": 256, "Q3_K": 256, "Q4_K": 256, "Q5_K": 256, "Q6_K": 256, "Q8_K": 256}
BYTES = {"Q8_0": 34, "Q2_K": 84, "Q3_K": 110, "Q4_K": 144, "Q5_K": 176, "Q6_K": 210, "Q8_K": 292}
TYPES = ("Q8_0", "Q2_K", "Q3_K", "Q4_K", "Q5_K", "Q6_K")
EPS = 1e-5

# Bounds of a drawn case, those of the largest listed ones.
MAX_NORM = 2048 * 4096
MAX_ROUTE = 512 * 128 * 2048
MAX_BYTES = 7.9e8  # of weights that a pass reads
MAX_WEIGHTS = 8 * 14336 * 4096
MAX_PAIRS = 64


def listed():
    return [
        # one token between two layers of an 8B model: f32 for the router, Q8_K for the experts
        {"name": "norm_q8k_1x4096", "kind": "norm", "tokens": 1, "cols": 4096, "packed": "Q8_K", "residual": True},
        # an odd prompt through a 0.5B model's norm, for Q8_0 weights
        {"name": "norm_q8_0_333x896", "kind": "norm", "tokens": 333, "cols": 896, "packed": "Q8_0", "residual": True},
        # a long prompt, the first norm of a model: nothing to add yet
        {"name": "norm_q8k_2048x4096", "kind": "norm", "tokens": 2048, "cols": 4096, "packed": "Q8_K", "residual": False},
        # one token's experts, two of eight
        {"name": "route_1x4096_2of8", "kind": "route", "tokens": 1, "cols": 4096, "experts": 8, "slots": 2,
         "gating": "softmax", "normalize": True, "bias": False},
        # an odd batch, sigmoid scores with a bias that balances the experts, some of them switched off
        {"name": "route_77x896_6of60_bias", "kind": "route", "tokens": 77, "cols": 896, "experts": 60, "slots": 6,
         "gating": "sigmoid", "normalize": True, "bias": True},
        # a prompt's experts, eight of 128
        {"name": "route_512x2048_8of128", "kind": "route", "tokens": 512, "cols": 2048, "experts": 128, "slots": 8,
         "gating": "softmax", "normalize": False, "bias": False},
        # one token through two of eight large experts, the down matrices in the larger type of a mixed file
        {"name": "ffn_q4k_1x8x14336x4096", "kind": "ffn", "tokens": 1, "experts": 8, "slots": 2, "cols": 4096,
         "ffn": 14336, "gate": "Q4_K", "down": "Q6_K", "packed": False, "residual": False, "dropped": 0.0},
        # one token through six of 64 small experts
        {"name": "ffn_q5k_1x64x1536x2048", "kind": "ffn", "tokens": 1, "experts": 64, "slots": 6, "cols": 2048,
         "ffn": 1536, "gate": "Q5_K", "down": "Q5_K", "packed": True, "residual": True, "dropped": 0.0},
        # five sequences decoded together, some of their places dropped, in a Q8_0 file with odd sizes
        {"name": "ffn_q8_0_5x16x1952x928", "kind": "ffn", "tokens": 5, "experts": 16, "slots": 4, "cols": 928,
         "ffn": 1952, "gate": "Q8_0", "down": "Q8_0", "packed": False, "residual": True, "dropped": 0.2},
        # a small batch of sequences through every large expert
        {"name": "ffn_q4k_32x8x14336x4096", "kind": "ffn", "tokens": 32, "experts": 8, "slots": 2, "cols": 4096,
         "ffn": 14336, "gate": "Q4_K", "down": "Q4_K", "packed": True, "residual": True, "dropped": 0.0},
        # the whole second half of a decoder layer for one token: norm, router and experts
        {"name": "layer_q4k_1x8x14336x4096", "kind": "layer", "tokens": 1, "experts": 8, "slots": 2, "cols": 4096,
         "ffn": 14336, "gate": "Q4_K", "down": "Q4_K"},
        # the same for eleven tokens and small experts in a smaller type
        {"name": "layer_q3k_11x32x1024x2048", "kind": "layer", "tokens": 11, "experts": 32, "slots": 4, "cols": 2048,
         "ffn": 1024, "gate": "Q3_K", "down": "Q2_K"},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _draw_layer(rng, kind):
    gate, down = rng.choice(TYPES), rng.choice(TYPES)
    experts = rng.choice((4, 8, 16, 40, 64))
    slots = rng.randint(1, min(experts, 8))
    # the norm's output serves the gate and up products, in blocks of their activations
    cols = BLOCK[gate] * _log(rng, max(1, 256 // BLOCK[gate]), 4096 // BLOCK[gate])
    ffn = BLOCK[down] * _log(rng, max(1, 256 // BLOCK[down]), 14336 // BLOCK[down])
    tokens = 1 if rng.random() < 0.4 else _log(rng, 2, 40)
    tokens = max(1, min(tokens, MAX_PAIRS // slots))
    case = {"kind": kind, "tokens": tokens, "experts": experts, "slots": slots, "cols": cols, "ffn": ffn, "gate": gate,
            "down": down}
    if kind == "ffn":
        case.update(packed=rng.random() < 0.5, residual=rng.random() < 0.5, dropped=rng.choice((0.0, 0.0, 0.3)))
    while experts * cols * case["ffn"] > MAX_WEIGHTS or work(case)["bytes"] > MAX_BYTES:
        case["ffn"] = BLOCK[down] * (case["ffn"] // (2 * BLOCK[down]))
    return case


def draw(rng):
    kind = rng.choices(("norm", "route", "ffn", "layer"), (25, 25, 35, 15))[0]
    if kind == "norm":
        packed = rng.choice(("Q8_K", "Q8_0"))
        cols = BLOCK[packed] * _log(rng, max(1, 128 // BLOCK[packed]), 14336 // BLOCK[packed])
        tokens = 1 if rng.random() < 0.25 else _log(rng, 2, max(2, min(4096, MAX_NORM // cols)))
        return {"kind": kind, "tokens": tokens, "cols": cols, "packed": packed, "residual": rng.random() < 0.6}
    if kind == "route":
        cols, experts = 32 * _log(rng, 8, 224), _log(rng, 2, 256)
        tokens = 1 if rng.random() < 0.25 else _log(rng, 2, max(2, min(1024, MAX_ROUTE // (cols * experts))))
        return {"kind": kind, "tokens": tokens, "cols": cols, "experts": experts, "slots": rng.randint(1, min(experts, 8)),
                "gating": rng.choice(("softmax", "sigmoid")), "normalize": rng.random() < 0.6, "bias": rng.random() < 0.4}
    return _draw_layer(rng, kind)


# ---- inputs ---------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=F32)


def _stream(gen, tokens, cols):
    """A residual stream: values of spread one, a few channels of them large."""
    loud = torch.rand((1, cols), generator=gen, device="cuda") < 0.005
    return _normal(gen, tokens, cols) * torch.where(loud, 12.0, 1.0)


def _levels(gen, n, lo, hi, sd, width=256):
    """[n, width] whole levels in lo..hi, normal about the middle."""
    x = torch.randn((n, width), generator=gen, device="cuda", dtype=F32)
    return x.mul_(sd).add_((lo + hi) / 2).round_().clamp_(lo, hi).to(torch.int16)


def _ints(gen, n, lo, hi, width):
    return torch.randint(lo, hi + 1, (n, width), generator=gen, device="cuda", dtype=torch.int16)


def _half(gen, n, middle):
    """[n, 1] f16 scales of 0.75 to 1.25 times `middle`."""
    u = torch.rand((n, 1), generator=gen, device="cuda", dtype=F32)
    return (u * 0.5 + 0.75).mul_(middle).to(torch.float16)


def _fields(*parts):
    """Blocks from their fields in order: whole numbers as bytes, or f16."""
    return torch.cat([p.view(torch.uint8) if p.dtype == torch.float16 else (p & 255).to(torch.uint8) for p in parts],
                     dim=1)


def _two_bits(q):
    """Levels 0..3 of 256 values: value 128h + 32s + j in bits 2s of byte 32h + j."""
    q = q.view(-1, 2, 4, 32)
    return (q[:, :, 0] | q[:, :, 1] << 2 | q[:, :, 2] << 4 | q[:, :, 3] << 6).reshape(-1, 64)


def _nibbles(q):
    """Levels 0..15 of 256 values: value 64g + j low, 64g + 32 + j high in byte 32g + j."""
    q = q.view(-1, 4, 2, 32)
    return (q[:, :, 0] | q[:, :, 1] << 4).reshape(-1, 128)


def _each(x, n):
    return x.repeat_interleave(n, dim=1)


def _blocks(t, n, gen, values):
    """n blocks of type t with weights of spread 0.02, and, if asked, the numbers
    they stand for, in 64 bits."""
    if t == "Q8_0":
        q, d = _levels(gen, n, -127, 127, 42.0, 32), _half(gen, n, 0.02 / 42)
        return _fields(d, q), d.to(F64) * q if values else None
    if t in ("Q4_K", "Q5_K"):
        top = 15 if t == "Q4_K" else 31
        q, sc = _levels(gen, n, 0, top, top / 4.4), _ints(gen, n, 20, 63, 8)
        mn = (sc.float() * (top / (top + 1.0))).round().to(torch.int16)
        d = _half(gen, n, 0.02 / (41.5 * top / 4.4))
        dmin = (d.float() * ((top + 1) / 2)).to(torch.float16)
        six = torch.cat([sc[:, :4] | (sc[:, 4:] >> 4) << 6, mn[:, :4] | (mn[:, 4:] >> 4) << 6,
                         (sc[:, 4:] & 15) | (mn[:, 4:] & 15) << 4], dim=1)
        fifth = (q >> 4).view(-1, 8, 32)
        high = [sum(fifth[:, s] << s for s in range(8))] if t == "Q5_K" else []
        w = d.to(F64) * (_each(sc, 32) * q) - dmin.to(F64) * _each(mn, 32) if values else None
        return _fields(d, dmin, six, *high, _nibbles(q & 15)), w
    if t == "Q6_K":
        q, d = _levels(gen, n, -32, 31, 13.0), _half(gen, n, 0.02 / (13 * 98))
        sc = _ints(gen, n, 70, 127, 16) * (_ints(gen, n, 0, 1, 16) * 2 - 1)
        u = (q + 32).view(-1, 2, 4, 32)
        ql = torch.stack([u[:, :, 0] & 15 | (u[:, :, 2] & 15) << 4, u[:, :, 1] & 15 | (u[:, :, 3] & 15) << 4], dim=2)
        return (_fields(ql.reshape(-1, 128), _two_bits((u >> 4).reshape(-1, 256)), sc, d),
                d.to(F64) * (_each(sc, 16) * q) if values else None)
    if t == "Q3_K":
        q, d = _levels(gen, n, -4, 3, 1.7), _half(gen, n, 0.02 / (1.7 * 24))
        sc = _ints(gen, n, 16, 31, 16) * (_ints(gen, n, 0, 1, 16) * 2 - 1)
        u, s = q + 4, sc + 32
        third = (u >> 2).view(-1, 8, 32)
        top = (s >> 4).view(-1, 4, 4)
        six = torch.cat([s[:, :8] & 15 | (s[:, 8:] & 15) << 4,
                         top[:, 0] | top[:, 1] << 2 | top[:, 2] << 4 | top[:, 3] << 6], dim=1)
        return (_fields(sum(third[:, k] << k for k in range(8)), _two_bits(u & 3), six, d),
                d.to(F64) * (_each(sc, 16) * q) if values else None)
    q, sc = _levels(gen, n, 0, 3, 0.9), _ints(gen, n, 7, 15, 16)  # Q2_K
    d = _half(gen, n, 0.02 / (0.9 * 11))
    dmin = (d.float() * 1.5).to(torch.float16)
    w = d.to(F64) * (_each(sc, 16) * q) - dmin.to(F64) * _each(sc, 16) if values else None
    return _fields(sc | sc << 4, _two_bits(q), d, dmin), w


def _matrices(t, n, rows, cols, gen, values=False):
    """n matrices of rows x cols: blocks [n, rows, cols / block, bytes], and their numbers."""
    b, w = _blocks(t, n * rows * cols // BLOCK[t], gen, values)
    return b.view(n, rows, cols // BLOCK[t], BYTES[t]), w.view(n, rows, cols) if values else None


def _chosen(case, gen):
    """Distinct experts of each token and their weights; dropped places hold -1."""
    chance = torch.rand((case["tokens"], case["experts"]), generator=gen, device="cuda")
    best = chance.topk(case["slots"], dim=1)
    weights = best.values / best.values.sum(1, keepdim=True)
    gone = torch.rand(weights.shape, generator=gen, device="cuda") < case["dropped"]
    ids = torch.where(gone, -1, best.indices).to(I32)
    return ids.contiguous(), weights.contiguous()


def _act(t):
    return "Q8_0" if t == "Q8_0" else "Q8_K"


def _inputs(case, seed, values=False):
    gen, kind = _generator(seed), case["kind"]
    T, K = case["tokens"], case["cols"]
    s = {"case": case}
    if kind in ("norm", "layer"):
        s["x"], s["norm"] = _stream(gen, T, K), _normal(gen, K) * 0.05 + 1.0
        s["residual"] = _stream(gen, T, K) if case.get("residual", True) else None
    if kind in ("route", "layer"):
        s["router"] = _normal(gen, case["experts"], K) * 0.03
    if kind == "route":
        s["x"] = _normal(gen, T, K)
        s["bias"] = None
        if case["bias"]:  # a learned balance; one expert of twelve is switched off
            off = torch.rand(case["experts"], generator=gen, device="cuda") < 1 / 12
            off[0] = False
            s["bias"] = torch.where(off, float("-inf"), _normal(gen, case["experts"]) * 0.2)
    if kind in ("ffn", "layer"):
        E, F = case["experts"], case["ffn"]
        for name, t, rows, cols in (("gate", case["gate"], F, K), ("up", case["gate"], F, K), ("down", case["down"], K, F)):
            s[name], s[name + "_values"] = _matrices(t, E, rows, cols, gen, values)
    if kind == "ffn":
        s["ids"], s["weights"] = _chosen(case, gen)
        s["x"] = _normal(gen, T, K)
        s["residual"] = _stream(gen, T, K) if case["residual"] else None
        if case["packed"]:
            s["x"] = _pack(_act(case["gate"]), s["x"])
    return s


# ---- the plain form ---------------------------------------------------------------

def _quantize(t, y):
    """Levels [.., blocks, block] and scales [.., blocks, 1] of f32 rows in Q8_K or
    Q8_0 blocks, each f32 operation of the format's definition rounded once."""
    v = y.reshape(*y.shape[:-1], -1, BLOCK[t])
    if t == "Q8_0":
        d = v.abs().amax(-1, keepdim=True)
        d = d / torch.full_like(d, 127.0)  # (a plain number's reciprocal would be multiplied by)
        inverse = torch.where(d != 0, 1.0 / d, 0.0)
        r = (v * inverse).to(F64)  # (half away from zero; the sum with a half is exact in 64 bits)
        q = (r.abs() + 0.5).floor().clamp(max=127).to(F32) * v.sign()
        return q, d.to(torch.float16).to(F32)
    first = v.abs().argmax(-1, keepdim=True)  # (the first of equal ones)
    top = v.gather(-1, first)
    inverse = torch.full_like(top, -127.0) / top
    zero = top == 0
    q = torch.where(zero, 0.0, (v * inverse).round().clamp(max=127))
    return q, torch.where(zero, 0.0, 1.0 / inverse)


def _pack(t, y):
    """GGUF bytes [tokens, bytes] of f32 rows in Q8_K or Q8_0 blocks."""
    q, d = _quantize(t, y)
    if t == "Q8_0":
        return _fields(d.reshape(-1, 1).to(torch.float16), q.reshape(-1, 32).to(torch.int16)).reshape(y.shape[0], -1)
    sums = q.reshape(-1, 16, 16).sum(-1).to(torch.int16)
    parts = [d.reshape(-1, 1).contiguous().view(torch.uint8), (q.reshape(-1, 256).to(torch.int16) & 255).to(torch.uint8),
             sums.view(torch.uint8)]
    return torch.cat(parts, dim=1).reshape(y.shape[0], -1)


def _unpack(t, b):
    """The numbers that rows of Q8_K or Q8_0 blocks stand for."""
    b = b.view(b.shape[0], -1, BYTES[t])
    if t == "Q8_0":
        d, q = b.view(torch.float16)[..., :1].to(F32), b[..., 2:]
    else:
        d, q = b.view(F32)[..., :1], b[..., 4:260]
    return (q.view(torch.int8) * d).reshape(b.shape[0], -1)


def _plain_norm(x, residual, weight, packed):
    total = x if residual is None else x + residual
    mean = (total * total).to(F64).sum(-1, keepdim=True) / total.shape[-1]
    y = total * (1.0 / (mean.to(F32) + EPS).sqrt()) * weight
    return total, y, _quantize(packed, y)


def _plain_route(case, x, router, bias):
    logits = (x.to(F64) @ router.to(F64).t()).to(F32)
    z = logits.to(F64)
    if case.get("gating", "softmax") == "softmax":
        e = (z - z.amax(1, keepdim=True)).exp()
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + (-z).exp())
    rank = z if bias is None else score + bias.to(F64)
    order = rank.argsort(dim=1, descending=True, stable=True)[:, :case["slots"]]
    none = rank.gather(1, order) == float("-inf")  # fewer experts than places
    chosen = torch.where(none, 0.0, score.gather(1, order))
    if case.get("normalize", True):
        chosen = chosen / chosen.sum(1, keepdim=True)
    return logits, torch.where(none, -1, order).to(I32), chosen.to(F32)


def _decode(t, b):
    """Blocks [.., bytes] as the numbers they stand for, [.., block], in 64 bits."""
    half = lambda i: b[..., i:i + 2].contiguous().view(torch.float16).to(F64)  # noqa: E731
    signed = lambda x: x.contiguous().view(torch.int8)  # noqa: E731
    flat = lambda x, n: x.reshape(*b.shape[:-1], n)  # noqa: E731
    if t == "Q8_0":
        return signed(b[..., 2:]) * half(0)
    if t in ("Q4_K", "Q5_K"):
        sc, mn, mix = b[..., 4:8], b[..., 8:12], b[..., 12:16]
        scale = torch.cat([sc & 63, mix & 15 | (sc >> 6) << 4], -1).to(F64) * half(0)
        low = torch.cat([mn & 63, mix >> 4 | (mn >> 6) << 4], -1).to(F64) * half(2)
        at = 16 if t == "Q4_K" else 48
        q = b[..., at:].reshape(*b.shape[:-1], 4, 1, 32)
        q = flat(torch.cat([q & 15, q >> 4], -2), 256)
        if t == "Q5_K":
            bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(8, 1)
            q = q + flat((b[..., None, 16:48] >> bit & 1) << 4, 256)
        return flat(q.reshape(*b.shape[:-1], 8, 32) * scale[..., None] - low[..., None], 256)
    two = torch.tensor([0, 2, 4, 6], device=b.device, dtype=torch.uint8).view(4, 1)
    if t == "Q6_K":
        ql = b[..., :128].reshape(*b.shape[:-1], 2, 1, 64)
        low = torch.cat([ql & 15, ql >> 4], -2).reshape(*b.shape[:-1], 2, 4, 32)
        high = b[..., 128:192].reshape(*b.shape[:-1], 2, 1, 32) >> two & 3
        scale = signed(b[..., 192:208]).to(F64) * half(208)
        return flat(((low | high << 4).to(torch.int16) - 32).reshape(*b.shape[:-1], 16, 16) * scale[..., None], 256)
    if t == "Q3_K":
        low = flat(b[..., 32:96].reshape(*b.shape[:-1], 2, 1, 32) >> two & 3, 256)
        bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(8, 1)
        high = flat(b[..., None, :32] >> bit & 1, 256)
        s = b[..., 96:104]
        top = (b[..., None, 104:108] >> two & 3).reshape(*b.shape[:-1], 16)
        six = torch.cat([s & 15, s >> 4], -1) | top << 4
        scale = (six.to(torch.int16) - 32).to(F64) * half(108)
        return flat(((low | high << 2).to(torch.int16) - 4).reshape(*b.shape[:-1], 16, 16) * scale[..., None], 256)
    sc = b[..., :16]  # Q2_K
    q = (b[..., 16:80].reshape(*b.shape[:-1], 2, 1, 32) >> two & 3).reshape(*b.shape[:-1], 16, 16)
    return flat(q * ((sc & 15).to(F64) * half(80))[..., None] - ((sc >> 4).to(F64) * half(82))[..., None], 256)


def _products(t, blocks, a, token, expert):
    """Pair p's product of matrix expert[p] with column token[p] of a, in 64 bits
    [pairs, rows].  Few pairs take their own matrices, many all of them."""
    if expert.numel() < blocks.shape[0]:
        w = _decode(t, blocks[expert]).flatten(2)
        return (w @ a[token].unsqueeze(-1)).squeeze(-1)
    w = _decode(t, blocks).flatten(2)
    y = (w.flatten(0, 1) @ a.t().contiguous()).view(w.shape[0], w.shape[1], a.shape[0])
    return y[expert, :, token]


def _plain_ffn(case, a, s, ids, weights, residual):
    T, S = ids.shape
    token = torch.arange(T, device=ids.device).repeat_interleave(S)
    expert = ids.reshape(-1).clamp(min=0).long()
    g = _products(case["gate"], s["gate"], a, token, expert).to(F32).to(F64)
    u = _products(case["gate"], s["up"], a, token, expert).to(F32).to(F64)
    h = (g / (1 + (-g).exp()) * u).to(F32)
    q, d = _quantize(_act(case["down"]), h)
    h = (q.to(F64) * d.to(F64)).flatten(1)
    y = _products(case["down"], s["down"], h, torch.arange(T * S, device=ids.device), expert)
    w = torch.where(ids >= 0, weights, 0.0).to(F64)
    y = (y.view(T, S, -1) * w.unsqueeze(-1)).sum(1)
    return (y if residual is None else y + residual.to(F64)).to(F32)


def _values(t, q, d):
    """Levels and scales as the numbers they stand for."""
    return (q.to(F64) * d.to(F64)).flatten(-2)


# ---- the protocol -------------------------------------------------------------------

_kept = {}


def _framework():
    if not _kept:
        _kept["rlq"] = importlib.import_module("rust-llama_amd")
        _kept["ctx"] = _kept["rlq"].Context(0)
    return _kept["rlq"], _kept["ctx"]


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] in ("ffn", "layer"):  # the weights as a program keeps them on the GPU
        rlq, ctx = _framework()
        for name, t, rows, cols in (("gate", case["gate"], case["ffn"], case["cols"]),
                                    ("up", case["gate"], case["ffn"], case["cols"]),
                                    ("down", case["down"], case["cols"], case["ffn"])):
            s[name] = rlq.Weights(ctx, rlq.DType[t], s[name].reshape(-1), rows, cols, case["experts"])
    return s


def _run_own(s):
    case, (rlq, ctx) = s["case"], _framework()
    kind = case["kind"]
    if kind == "norm":
        total, y, q = ctx.rms_norm(s["x"], s["norm"], EPS, residual=s["residual"], packed=rlq.DType[case["packed"]])
        return {"total": total, "y": y, "packed": _unpack(case["packed"], q)}
    if kind == "route":
        ids, weights, logits = ctx.moe_route(s["router"], s["x"], case["slots"], gating=case["gating"],
                                             normalize=case["normalize"], bias=s["bias"], logits=True)
        return {"ids": ids, "weights": weights, "logits": logits}
    act = rlq.DType[_act(case["gate"])]
    if kind == "ffn":
        return ctx.moe_ffn(s["gate"], s["up"], s["down"], s["x"], s["ids"], s["weights"],
                           x_dtype=act if case["packed"] else rlq.DType.F32, residual=s["residual"])
    total, y, q = ctx.rms_norm(s["x"], s["norm"], EPS, residual=s["residual"], packed=act)
    ids, weights, _ = ctx.moe_route(s["router"], y, case["slots"])
    out = ctx.moe_ffn(s["gate"], s["up"], s["down"], q, ids, weights, x_dtype=act, residual=total)
    return {"ids": ids, "weights": weights, "y": out}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        total, y, (q, d) = _plain_norm(s["x"], s["residual"], s["norm"], case["packed"])
        return {"total": None if s["residual"] is None else total, "y": y, "packed": (q * d).flatten(1)}
    if kind == "route":
        logits, ids, weights = _plain_route(case, s["x"], s["router"], s["bias"])
        return {"ids": ids, "weights": weights, "logits": logits}
    act = _act(case["gate"])
    if kind == "ffn":
        a = _unpack64(act, s["x"]) if case["packed"] else _values(act, *_quantize(act, s["x"]))
        return _plain_ffn(case, a, s, s["ids"], s["weights"], s["residual"])
    total, y, (q, d) = _plain_norm(s["x"], s["residual"], s["norm"], act)
    _, ids, weights = _plain_route(case, y, s["router"], None)
    return {"ids": ids, "weights": weights, "y": _plain_ffn(case, _values(act, q, d), s, ids, weights, total)}


def _unpack64(t, b):
    """The numbers that rows of Q8_K or Q8_0 blocks stand for, in 64 bits."""
    b = b.view(b.shape[0], -1, BYTES[t])
    at, kind = (2, torch.float16) if t == "Q8_0" else (4, F32)
    d, q = b[..., :at].contiguous().view(kind).to(F64), b[..., at:at + BLOCK[t]]
    return (q.contiguous().view(torch.int8) * d).reshape(b.shape[0], -1)


def work(case):
    kind, T, K = case["kind"], case["tokens"], case["cols"]
    norm = T * K * (4 * (1 + 2 * case.get("residual", True)) + 4) + K * 4
    if kind == "norm":
        return {"bytes": norm + T * K // BLOCK[case["packed"]] * BYTES[case["packed"]], "flops": 8.0 * T * K}
    E, S = case["experts"], case["slots"]
    route = {"bytes": 4 * (E * K + T * K + 2 * T * S), "flops": 2.0 * T * E * K}
    if kind == "route":
        return {"bytes": route["bytes"] + 4 * T * E + 4 * E * case["bias"], "flops": route["flops"]}
    F, pairs = case["ffn"], T * S * (1 - case.get("dropped", 0.0))
    used = E * (1 - (1 - S * (1 - case.get("dropped", 0.0)) / E) ** T)  # experts that some token chose, expected
    weights = 2 * F * K // BLOCK[case["gate"]] * BYTES[case["gate"]] + K * F // BLOCK[case["down"]] * BYTES[case["down"]]
    act = K // BLOCK[_act(case["gate"])] * BYTES[_act(case["gate"])] if case.get("packed") else 4 * K
    ffn = {"bytes": used * weights + T * (act + 4 * K * (1 + case.get("residual", True)) + 8 * S),
           "flops": 6.0 * pairs * F * K}
    if kind == "ffn":
        return ffn
    return {"bytes": ffn["bytes"] - T * (act + 4 * K) + route["bytes"] - 4 * T * K + 8 * T * K + 4 * K,
            "flops": ffn["flops"] + route["flops"] + 8.0 * T * K}


# ---- the definition in 64 bits ----------------------------------------------------------

def _once(x):
    """A 64-bit number where the definition makes an f32 of it."""
    return x.to(F32).to(F64)


def _exact_blocks(t, y):
    """f32 rows (held in 64 bits) as the numbers of their 8-bit blocks."""
    b = y.reshape(-1, BLOCK[t])
    if t == "Q8_0":
        d = _once(b.abs().amax(1, keepdim=True) / 127)
        v = _once(b * torch.where(d > 0, _once(1 / d), 0.0))
        # |v| <= 127, so every v and v + 1/2 is exact here
        return (v.sign() * (v.abs() + 0.5).floor() * d.to(torch.float16).to(F64)).reshape(y.shape)
    hi, lo = b.max(1, keepdim=True), b.min(1, keepdim=True)
    up = (hi.values > -lo.values) | ((hi.values == -lo.values) & (hi.indices < lo.indices))
    inverse = _once(-127 / torch.where(up, hi.values, lo.values))
    v = _once(b * inverse).round() * _once(1 / inverse)
    return torch.where((hi.values == 0) & (lo.values == 0), 0.0, v).reshape(y.shape)


def _exact_norm(s):
    x = s["x"].to(F64)
    x = x if s["residual"] is None else _once(x + s["residual"].to(F64))
    mean = _once(_once(x * x).mean(1, keepdim=True))
    scale = _once(1 / _once(_once(mean + float(torch.tensor(EPS, dtype=F32))).sqrt()))
    return x, _once(_once(x * scale) * s["norm"].to(F64))


def _exact_route(case, x, s):
    z = _once((x.unsqueeze(1) * s["router"].to(F64)).sum(-1) if x.shape[0] == 1 else x @ s["router"].to(F64).t())
    score = torch.softmax(z, 1) if case.get("gating", "softmax") == "softmax" else torch.sigmoid(z)
    bias = s.get("bias")
    rank = z.clone() if bias is None else score + bias.to(F64)
    ids, weights = [], []
    for _ in range(case["slots"]):  # the best one left, the lowest index of equal ones
        top = rank.amax(1, keepdim=True)
        best, some = (rank == top).to(torch.uint8).argmax(1, keepdim=True), top > float("-inf")
        ids.append(torch.where(some, best, -1))
        weights.append(score.gather(1, best) * some)
        rank.scatter_(1, best, float("-inf"))
    ids, weights = torch.cat(ids, 1), torch.cat(weights, 1)
    return z, ids, weights / weights.sum(1, keepdim=True) if case.get("normalize", True) else weights


def _exact_ffn(case, a, s, ids, weights, residual):
    y = torch.zeros((ids.shape[0], case["cols"]), dtype=F64, device="cuda") if residual is None else residual.clone()
    for e in range(case["experts"]):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if not token.numel():
            continue
        g, u = (_once(a[token] @ s[name + "_values"][e].t()) for name in ("gate", "up"))
        h = _exact_blocks(_act(case["down"]), _once(g * torch.sigmoid(g) * u))
        y.index_add_(0, token, h @ s["down_values"][e].t() * weights[token, slot].to(F64).unsqueeze(1))
    return y


def exact(case, seed):
    s = _inputs(case, seed, values=True)
    kind = case["kind"]
    if kind == "norm":
        total, y = _exact_norm(s)
        return {"total": None if s["residual"] is None else total, "y": y, "packed": _exact_blocks(case["packed"], y)}
    if kind == "route":
        z, ids, weights = _exact_route(case, s["x"].to(F64), s)
        return {"ids": ids, "weights": weights, "logits": z}
    act = _act(case["gate"])
    if kind == "ffn":
        a = _unpack64(act, s["x"]) if case["packed"] else _exact_blocks(act, s["x"].to(F64))
        return _exact_ffn(case, a, s, s["ids"], s["weights"], None if s["residual"] is None else s["residual"].to(F64))
    total, y = _exact_norm(s)
    _, ids, weights = _exact_route(case, y, s)
    weights = _once(weights)
    return {"ids": ids, "weights": weights, "y": _exact_ffn(case, _exact_blocks(act, y), s, ids, weights, total)}
