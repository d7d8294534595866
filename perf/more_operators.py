"""Serving several requests from one paged KV cache, and beam search over it: what
is measured, and what it is compared with.

Five operators of `Context`:

  kv_pages      the requests' lengths turned into pages off a free list, block
                tables, the slot, position and request of every new token
  kv_store      queries and keys rotated by their positions, keys and values
                written to their slots (f32, f16, bf16 or Q8_0)
  kv_attention  one new token's query heads over its request's pages
  beam_select   the best continuations of a group of beams over the vocabulary
  beam_reorder  the beams' block tables after that choice, and the pages that are
                only partly filled

`run` computes them in torch's elementary operations, or, where `own` is set, by
the framework's calls.

Rotations are angles and products in 64 bits, rounded to f32 once, so that a cache's
16-bit values and 8-bit levels are defined to the last one; beams are ranked in 64
bits; attention is f32.
"""
import importlib

import numpy as np
import torch

own = False  # True: `run` makes the framework's calls

F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
KINDS = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
SIZE = {"F32": 4.0, "F16": 2.0, "BF16": 2.0, "Q8_0": 34 / 32}
NONE = float("-inf")

# Bounds of a drawn case, those of the largest listed ones.
MAX_TOKENS = 65536
MAX_STORE = 1777 * 24 * 128
MAX_READ = 5.4e8
MAX_LOGITS = 16 * 8 * 151936
MAX_COPY = 8 * 8 * 16 * 8 * 64 * 128


def listed():
    return [
        # a decode step's bookkeeping: one more token for each of 32 requests, some of them ended
        {"name": "pages_32_decode", "kind": "pages", "requests": 32, "context": 8192, "new": 1, "budget": 32, "page": 16,
         "ended": 0.1},
        # prompts of all lengths come in, as many as the batch has room for
        {"name": "pages_256_prompts", "kind": "pages", "requests": 256, "context": 4096, "new": 2000, "budget": MAX_TOKENS,
         "page": 32, "ended": 0.1},
        # one token of an 8B model
        {"name": "store_f16_1x32x8x128", "kind": "store", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128,
         "pairs": True, "type": "F16", "page": 16, "start": 1000},
        # an odd prompt of a 0.5B model into an 8-bit cache, far into a long context
        {"name": "store_q8_0_1777x14x2x64", "kind": "store", "tokens": 1777, "heads": 14, "kv_heads": 2, "dim": 64,
         "rotated": 64, "pairs": False, "type": "Q8_0", "page": 32, "start": 100000},
        # one sequence of an 8B model at a middling context
        {"name": "attn_f16_1x1000", "kind": "attn", "requests": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "F16", "page": 16, "longest": 1000, "even": True, "window": 0, "empty": 0.0, "padding": 0},
        # the same at a very long one
        {"name": "attn_bf16_1x131072", "kind": "attn", "requests": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "BF16", "page": 64, "longest": 131072, "even": True, "window": 0, "empty": 0.0, "padding": 0},
        # 32 requests of all lengths decoded together
        {"name": "attn_f16_32x8192", "kind": "attn", "requests": 32, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "F16", "page": 16, "longest": 8192, "even": False, "window": 0, "empty": 0.0, "padding": 0},
        # an odd batch of a 0.5B model in an 8-bit cache that looks back 1000 tokens, a captured batch's rows behind it
        {"name": "attn_q8_0_77x5000_window", "kind": "attn", "requests": 77, "tokens": 1, "heads": 14, "kv_heads": 2,
         "dim": 64, "type": "Q8_0", "page": 32, "longest": 5000, "even": False, "window": 1000, "empty": 0.1, "padding": 3},
        # four beams of one request over an 8B model's vocabulary
        {"name": "select_1x4x128256_8", "kind": "select", "groups": 1, "beams": 4, "vocabulary": 128256, "best": 8},
        # eight beams for each of 16 requests over a 0.5B model's vocabulary
        {"name": "select_16x8x151936_16", "kind": "select", "groups": 16, "beams": 8, "vocabulary": 151936, "best": 16},
        # one request's beams in two layers
        {"name": "reorder_1x4_2layers", "kind": "reorder", "groups": 1, "beams": 4, "layers": 2, "kv_heads": 8, "dim": 128,
         "type": "F16", "page": 16, "length": 1000},
        # eight requests' beams in eight layers with larger pages
        {"name": "reorder_8x8_8layers", "kind": "reorder", "groups": 8, "beams": 8, "layers": 8, "kv_heads": 8, "dim": 128,
         "type": "BF16", "page": 64, "length": 1977},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choices(("pages", "store", "attn", "select", "reorder"), (15, 20, 35, 15, 15))[0]
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "pages":
        requests = _log(rng, 1, 512)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 4000)
        budget = requests if new == 1 else _log(rng, 64, MAX_TOKENS)
        return {"kind": kind, "requests": requests, "context": _log(rng, 1, 16384), "new": new, "budget": budget, "page": page,
                "ended": rng.choice((0.0, 0.1, 0.3))}
    if kind == "select":
        vocabulary = _log(rng, 500, 151936)
        beams = _log(rng, 1, 16)
        groups = _log(rng, 1, max(1, min(64, MAX_LOGITS // (vocabulary * beams))))
        return {"kind": kind, "groups": groups, "beams": beams, "vocabulary": vocabulary, "best": rng.randint(1, 2 * beams)}
    dim, kv_heads = rng.choice((32, 64, 96, 128, 192, 256)), rng.choice((1, 2, 3, 4, 8))
    stored = rng.choice(("F32", "F16", "F16", "BF16", "BF16", "Q8_0", "Q8_0"))
    heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 16))
    if kind == "store":
        per = (heads + 2 * kv_heads) * dim
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, max(2, min(4096, MAX_STORE // per)))
        return {"kind": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotated": rng.choice((dim, dim, dim // 2)), "pairs": rng.random() < 0.5, "type": stored, "page": page,
                "start": _log(rng, 1, 1000000)}
    if kind == "reorder":
        beams, layers = rng.randint(2, 16), _log(rng, 1, 16)
        copied = beams * 2 * layers * kv_heads * page * dim
        return {"kind": kind, "groups": _log(rng, 1, max(1, min(32, MAX_COPY // copied))), "beams": beams, "layers": layers,
                "kv_heads": kv_heads, "dim": dim, "type": stored, "page": page, "length": _log(rng, 1, 8192)}
    requests = 1 if rng.random() < 0.25 else _log(rng, 2, 128)
    most = int(MAX_READ / (requests * kv_heads * dim * 2 * 4))  # (the plain form holds f32 copies)
    return {"kind": kind, "requests": requests, "tokens": rng.choice((1, 1, 1, 2, 5)), "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "type": stored, "page": page, "longest": _log(rng, 1, max(1, min(131072, most))),
            "even": rng.random() < 0.3, "window": rng.choice((0, 0, 0, 1, 100, 4096)), "empty": rng.choice((0.0, 0.0, 0.2)),
            "padding": rng.choice((0, 0, 5))}


# ---- inputs ---------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=F32)


def _lengths(gen, n, lo, hi):
    """n whole numbers spread over the logarithm of lo..hi (lo >= 1)."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=F64)
    return (lo * (hi / lo) ** u).round().clamp(lo, hi).to(I64)


def _shuffled(gen, n):
    return torch.randperm(n, generator=gen, device="cuda")


def _bytes_of(levels, scales):
    """A Q8_0 cache [.., page * (dim + dim / 16)] uint8: a head's levels in a page, token after token, then their scales."""
    return torch.cat([levels.to(torch.int8).view(torch.uint8).flatten(-2), scales.view(torch.uint8).flatten(-2)], -1)


def _split(b, page, dim):
    """Views of a Q8_0 cache: levels [.., page, dim] int8 and scales [.., page, dim / 32] f16."""
    levels = b[..., :page * dim].view(torch.int8).unflatten(-1, (page, dim))
    return levels, b[..., page * dim:].view(torch.float16).unflatten(-1, (page, dim // 32))


def _cache(gen, case, *shape):
    """Random contents of a cache [.., page, dim]."""
    page, dim = case["page"], case["dim"]
    if case["type"] == "Q8_0":
        q = torch.randint(-127, 128, (*shape, page, dim), generator=gen, device="cuda", dtype=torch.int8)
        u = torch.rand((*shape, page, dim // 32), generator=gen, device="cuda", dtype=F32)
        return _bytes_of(q, (u * 0.5 + 0.75).mul_(1 / 64).to(torch.float16))
    return torch.randn((*shape, page, dim), generator=gen, device="cuda", dtype=KINDS[case["type"]])


def _inputs_pages(case, gen):
    n, page = case["requests"], case["page"]
    before = _lengths(gen, n, 1, case["context"])
    before[torch.rand(n, generator=gen, device="cuda") < 0.2] = 0  # requests that have just come
    new = _lengths(gen, n, 1, case["new"])
    new = torch.minimum(new, (case["budget"] - new.cumsum(0) + new).clamp(min=0))  # (the last ones have to wait)
    new[torch.rand(n, generator=gen, device="cuda") < case["ended"]] = -1
    wide = -(-(case["context"] + case["new"]) // page)
    pool = n * wide
    held = -(-before // page)
    first = held.cumsum(0) - held
    column = torch.arange(wide, device="cuda")
    order = _shuffled(gen, pool)
    tables = torch.where(column < held[:, None], order[(first[:, None] + column).clamp(max=pool - 1)], -1).to(I32)
    used = held.sum()
    free = order[(torch.arange(pool, device="cuda") + used).clamp(max=pool - 1)].to(I32)
    return {"before": before.to(I32), "new": new.to(I32), "tables": tables.contiguous(), "free": free,
            "count": (pool - used).to(I32).reshape(1), "tokens": case["budget"]}


def _inputs_store(case, gen):
    T, H, K, D, page = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page"))
    fused = _normal(gen, T, (H + 2 * K) * D)  # one product makes the three
    pages = -(-T // page) + 5
    position = torch.arange(T, device="cuda") + case["start"]
    order = _shuffled(gen, pages)
    at = torch.arange(T, device="cuda") + case["start"] % page
    pages_needed = order[(at // page) % pages]
    half = case["rotated"] // 2
    freqs = 500000.0 ** (-torch.arange(half, device="cuda", dtype=F64) / half)
    return {"q": fused[:, :H * D].unflatten(1, (H, D)), "k": fused[:, H * D:(H + K) * D].unflatten(1, (K, D)),
            "v": fused[:, (H + K) * D:].unflatten(1, (K, D)), "slots": pages_needed * page + at % page,
            "positions": position.to(I32), "freqs": freqs.to(F32), "kc": _cache(gen, case, pages, K),
            "vc": _cache(gen, case, pages, K)}


def _inputs_attn(case, gen):
    R, each, H, K, D, page = (case[k] for k in ("requests", "tokens", "heads", "kv_heads", "dim", "page"))
    wide = -(-case["longest"] // page)
    length = torch.full((R,), case["longest"], device="cuda") if case["even"] else _lengths(gen, R, 1, case["longest"])
    length[0] = case["longest"]
    tables = _shuffled(gen, R * wide).to(I32).view(R, wide)
    rows = R * each
    back = torch.arange(each - 1, -1, -1, device="cuda")
    positions = (length[:, None] - 1 - back).clamp(min=-1).reshape(-1)  # the last tokens of each request
    positions[torch.rand(rows, generator=gen, device="cuda") < case["empty"]] = -1
    requests = torch.arange(R, device="cuda").repeat_interleave(each)
    if case["padding"]:
        behind = torch.full((case["padding"],), -1, device="cuda")
        positions, requests = torch.cat([positions, behind]), torch.cat([requests, behind])
    return {"q": _normal(gen, rows + case["padding"], H, D), "tables": tables, "positions": positions.to(I32),
            "requests": requests.to(I32), "out": _normal(gen, rows + case["padding"], H, D),
            "kc": _cache(gen, case, R * wide, K), "vc": _cache(gen, case, R * wide, K)}


def _inputs_select(case, gen):
    G, B, V = case["groups"], case["beams"], case["vocabulary"]
    z = _normal(gen, G, B, V) * 2.5
    z[torch.rand((G, B, V), generator=gen, device="cuda") < 0.01] = NONE  # tokens that may not follow
    scores = -20 * torch.rand((G, B), generator=gen, device="cuda")
    dead = torch.rand((G, B), generator=gen, device="cuda") < 0.1  # beams that have no place any more
    dead[:, 0] = False
    return {"logits": z, "scores": torch.where(dead, NONE, scores)}


def _inputs_reorder(case, gen):
    G, B, page = case["groups"], case["beams"], case["page"]
    wide, pool = -(-(case["length"] + 64) // page), 2 * G * B + 64
    # whole pages may be anybody's; the page that is being filled is a beam's own
    tables = torch.randint(0, pool, (G * B, wide), generator=gen, device="cuda")
    tables[:, case["length"] // page] = _shuffled(gen, pool)[:G * B]
    best = torch.rand((G, B, B), generator=gen, device="cuda").square()  # a few parents have most of the children
    parents = (best * B).long().clamp(max=B - 1).amin(-1)
    parents[torch.rand((G, B), generator=gen, device="cuda") < 0.03] = -1  # no candidate was left
    return {"parents": parents.to(I32), "lengths": torch.full((G, B), case["length"], device="cuda", dtype=I32),
            "tables": tables.to(I32), "kv": _cache(gen, case, 2 * case["layers"], pool, case["kv_heads"])}


INPUTS = {"pages": _inputs_pages, "store": _inputs_store, "attn": _inputs_attn, "select": _inputs_select,
          "reorder": _inputs_reorder}


def _inputs(case, seed):
    s = INPUTS[case["kind"]](case, torch.Generator(device="cuda").manual_seed(seed))
    s["case"] = case
    return s


# ---- the plain forms -----------------------------------------------------------------

def _plain_pages(s):
    page, tables, free = s["case"]["page"], s["tables"], s["free"]
    before, new, n = s["before"].long(), s["new"].long(), s["count"].long()
    ended = new < 0
    more = new.clamp(min=0)
    after = torch.where(ended, 0, before + more)
    held, need = -(-before // page), -(-after // page)
    column = torch.arange(tables.shape[1], device=free.device)
    # the free list with the ended requests' pages on its top
    gone = (ended[:, None] & (column < held[:, None]) & (tables >= 0)).reshape(-1)
    at = torch.where(gone, n + gone.cumsum(0) - 1, free.numel())
    stack = torch.cat([free, free.new_zeros(1)]).scatter(0, at, tables.reshape(-1))
    top = n + gone.sum()
    # pages are taken off its top, a request after the other
    fresh = ~ended[:, None] & (column >= held[:, None]) & (column < need[:, None])
    turn = fresh.reshape(-1).cumsum(0).view(fresh.shape)
    taken = stack[torch.where(fresh, top - turn, 0)]
    tables.copy_(torch.where(fresh, taken, torch.where(gone.view(fresh.shape), -1, tables)))
    left = top - fresh.sum()
    place = torch.arange(free.numel(), device=free.device)
    free.copy_(torch.where((place >= n) & (place < top), stack[:-1], free))
    # the new tokens, a request after the other
    ends = more.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    token = torch.arange(s["tokens"], device=free.device)
    r = torch.searchsorted(ends, token, right=True)
    live, r = r < before.numel(), r.clamp(max=before.numel() - 1)
    position = torch.where(live, before[r] + token - starts[r], 0)
    slot = tables[r, position // page].long() * page + position % page
    return {"tables": tables, "free": free, "count": left.to(I32), "lengths": after.to(I32), "starts": starts.to(I32),
            "slots": torch.where(live, slot, -1), "positions": torch.where(live, position, -1).to(I32),
            "requests": torch.where(live, r, -1).to(I32)}


def _rotate(x, positions, freqs, pairs):
    """x [tokens, heads, dim] f32; the first 2 * freqs values of a head are rotated."""
    half = freqs.numel()
    angle = (positions.to(F64)[:, None] * freqs.to(F64))[:, None]
    c, s, y = angle.cos(), angle.sin(), x.to(F64)
    a, b = (y[..., :2 * half:2], y[..., 1:2 * half:2]) if pairs else (y[..., :half], y[..., half:2 * half])
    turned = torch.stack([a * c - b * s, a * s + b * c], -1) if pairs else torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned.flatten(2) if pairs else turned, y[..., 2 * half:]], -1).to(F32)


def _levels(y):
    """Levels [.., dim] and f16 scales [.., dim / 32] of f32 rows in Q8_0 blocks, each f32 operation rounded once."""
    v = y.unflatten(-1, (-1, 32))
    d = v.abs().amax(-1, keepdim=True)
    d = d / torch.full_like(d, 127.0)  # (a plain number's reciprocal would be multiplied by)
    r = (v * torch.where(d != 0, 1.0 / d, 0.0)).to(F64)  # (half away from zero; the sum with a half is exact in 64 bits)
    q = (r.abs() + 0.5).floor().clamp(max=127) * r.sign()
    return q.to(torch.int8).flatten(-2), d.squeeze(-1).to(torch.float16)


def _write(cache, case, slots, y):
    page = case["page"]
    p, o = slots // page, slots % page
    if case["type"] != "Q8_0":
        cache[p, :, o] = y.to(cache.dtype)
        return
    levels, scales = _split(cache, page, case["dim"])
    levels[p, :, o], scales[p, :, o] = _levels(y)


def _values(cache, case):
    """A cache as the numbers that it stands for, [.., page, dim] (f32, 16 bits as they are)."""
    if case["type"] != "Q8_0":
        return cache
    levels, scales = _split(cache, case["page"], case["dim"])
    return (levels.unflatten(-1, (-1, 32)).to(F32) * scales.to(F32).unsqueeze(-1)).flatten(-2)


def _plain_store(s):
    case = s["case"]
    q = _rotate(s["q"], s["positions"], s["freqs"], case["pairs"])
    _write(s["kc"], case, s["slots"], _rotate(s["k"], s["positions"], s["freqs"], case["pairs"]))
    _write(s["vc"], case, s["slots"], s["v"])
    return q


def _plain_attn(s):
    case = s["case"]
    H, K, D, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    R, wide = s["tables"].shape
    n, live = wide * page, s["requests"] >= 0
    rows = s["requests"].clamp(min=0).long().view(-1, 1)
    # every request's keys and values, [requests, kv heads, tokens, dim]
    k, v = (_values(c[s["tables"].long()], case).to(F32).transpose(1, 2).reshape(R, K, n, D) for c in (s["kc"], s["vc"]))
    each, R = case["tokens"], case["requests"]
    q = s["q"][:R * each].view(R, each, K, H // K, D).transpose(1, 2).reshape(R, K, -1, D) * D ** -0.5
    z = (q @ k.transpose(2, 3)).view(R, K, each, H // K, n)
    last, at = s["positions"][:R * each].view(R, 1, each, 1, 1), torch.arange(n, device=q.device)
    seen = at <= last
    if case["window"]:
        seen = seen & (at > last - case["window"])
    z = torch.where(seen, z, NONE)
    top = z.amax(-1, keepdim=True)
    p = torch.where(seen, (z - torch.where(top == NONE, 0.0, top)).exp(), 0.0)
    y = p.view(R, K, -1, n) @ v
    y = y.view(R, K, each, H // K, D) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"][:R * each] = y.transpose(1, 2).reshape(R * each, H, D)
    return s["out"]


def _plain_select(s):
    G, B, V = s["logits"].shape
    best = s["case"]["best"]
    z = s["logits"].to(F64)
    top = z.amax(-1, keepdim=True)
    total = (top + (z - top).exp().sum(-1, keepdim=True).log()).neg() + z + s["scores"].to(F64).unsqueeze(-1)
    total = torch.where(s["scores"].unsqueeze(-1) == NONE, NONE, total).view(G, B * V)
    order = total.argsort(dim=1, descending=True, stable=True)[:, :best]
    score = total.gather(1, order)
    none = score == NONE
    return {"scores": score.to(F32), "parents": torch.where(none, -1, order // V).to(I32),
            "tokens": torch.where(none, -1, order % V).to(I32)}


def _plain_reorder(s):
    case = s["case"]
    G, B = s["parents"].shape
    page, tail, n = case["page"], case["length"] // case["page"], case["length"] % case["page"]
    beam = torch.arange(G * B, device=s["tables"].device).view(G, B)
    source = torch.where(s["parents"] < 0, beam, beam - beam % B + s["parents"]).view(-1)
    mine, theirs = s["tables"][:, tail].long(), s["tables"][source, tail].long()
    whole = torch.arange(s["tables"].shape[1], device=beam.device) < tail
    s["tables"].copy_(torch.where(whole, s["tables"][source], s["tables"]))
    for part in _split(s["kv"], page, case["dim"]) if case["type"] == "Q8_0" else (s["kv"],):
        part[:, mine, :, :n] = part[:, theirs, :, :n]
    return {"tables": s["tables"], "kv": s["kv"]}


PLAIN = {"pages": _plain_pages, "store": _plain_store, "attn": _plain_attn, "select": _plain_select,
         "reorder": _plain_reorder}


# ---- the protocol -------------------------------------------------------------------

_kept = {}


def _framework():
    if not _kept:
        _kept["rlq"] = importlib.import_module("rust-llama_amd")
        _kept["ctx"] = _kept["rlq"].Context(0)
    return _kept["rlq"], _kept["ctx"]


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        if case["kind"] in ("store", "attn", "reorder"):  # the handles of the caches' layers
            rlq, _ = _framework()
            pairs = s["kv"].unflatten(0, (-1, 2)).unbind() if "kv" in s else [(s["kc"], s["vc"])]
            s["caches"] = [rlq.KvCache(k, v, rlq.DType[case["type"]], case["page"], case["dim"]) for k, v in pairs]
    return s


def _run_own(s):
    case, (_, ctx) = s["case"], _framework()
    kind = case["kind"]
    if kind == "pages":
        lengths, count, starts, slots, positions, requests = ctx.kv_pages(
            s["before"], s["new"], s["tables"], s["free"], s["count"], case["page"], s["tokens"])
        return {"tables": s["tables"], "free": s["free"], "count": count, "lengths": lengths, "starts": starts,
                "slots": slots, "positions": positions, "requests": requests}
    if kind == "store":
        return ctx.kv_store(s["caches"][0], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"],
                            freqs=s["freqs"], pairs=case["pairs"])
    if kind == "attn":
        return ctx.kv_attention(s["caches"][0], s["q"], s["tables"], s["positions"], requests=s["requests"],
                                window=case["window"], out=s["out"])
    if kind == "select":
        scores, parents, tokens = ctx.beam_select(s["logits"], s["scores"], case["best"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    ctx.beam_reorder(s["parents"], s["lengths"], s["tables"], s["caches"])
    return {"tables": s["tables"], "kv": s["kv"]}


def run(s):
    if own:
        out = _run_own(s)
    else:
        out = PLAIN[s["case"]["kind"]](s)
    if s["case"]["kind"] == "store":
        return {"q": out, "k": _values(s["kc"], s["case"]), "v": _values(s["vc"], s["case"])}
    if s["case"]["kind"] == "reorder":
        out["kv"] = _values(out["kv"], s["case"])
    return out


def work(case):
    kind = case["kind"]
    if kind == "pages":
        n = case["requests"]
        tokens = min(n * _mean(1, case["new"]), case["budget"]) * (1 - case["ended"])
        return {"bytes": 20 * n + 16 * case["budget"] + 8 * (tokens / case["page"] + 0.5 * n), "flops": 0.0}
    if kind == "select":
        n = case["groups"] * case["beams"] * case["vocabulary"]
        return {"bytes": 4.0 * n * 0.9 + 12 * case["groups"] * case["best"], "flops": 4.0 * n}
    K, D, size = case["kv_heads"], case["dim"], SIZE[case["type"]]
    if kind == "store":
        T, H = case["tokens"], case["heads"]
        return {"bytes": T * (4 * (2 * H + 2 * K) * D + 2 * K * D * size + 12), "flops": 3.0 * T * (H + K) * case["rotated"]}
    if kind == "reorder":
        G, B, n = case["groups"], case["beams"], case["length"] % case["page"]
        moved = G * B * 0.6  # (beams whose parent is another)
        return {"bytes": 2 * moved * 2 * case["layers"] * K * n * D * size + 8 * G * B * (case["length"] // case["page"] + 2),
                "flops": 0.0}
    R, each, H = case["requests"], case["tokens"], case["heads"]
    seen = case["longest"] if case["even"] else _mean(1, case["longest"])
    if case["window"]:
        seen = min(seen, case["window"])
    rows = R * each * (1 - case["empty"])
    return {"bytes": R * seen * 2 * K * D * size + 8.0 * rows * H * D + 4 * R * seen / case["page"],
            "flops": 4.0 * rows * seen * H * D}


def _mean(lo, hi):
    """The mean of numbers spread over the logarithm of lo..hi."""
    return lo if hi <= lo else (hi - lo) / float(np.log(hi / lo))


# ---- the definition in 64 bits ----------------------------------------------------------

def _exact_pages(s):
    page = s["case"]["page"]
    before, new, tables, free = (s[k].cpu().numpy().copy() for k in ("before", "new", "tables", "free"))
    stack = list(free[:int(s["count"])])
    n = len(stack)
    for r in np.flatnonzero(new < 0):
        held = -(-int(before[r]) // page)
        stack += [p for p in tables[r, :held] if p >= 0]
        tables[r, :held] = -1
    free[n:len(stack)] = stack[n:]
    after, starts, slots, positions, requests = [], [0], [], [], []
    for r in range(len(before)):
        have, end = int(before[r]), 0 if new[r] < 0 else int(before[r] + new[r])
        for j in range(-(-have // page), -(-end // page)):
            tables[r, j] = stack.pop()
        at = np.arange(have, end, dtype=np.int64)
        slots.append(tables[r, at // page].astype(np.int64) * page + at % page)
        positions.append(at)
        requests.append(np.full(len(at), r))
        after.append(end)
        starts.append(starts[-1] + len(at))
    rest = np.full(s["tokens"] - starts[-1], -1)
    to = lambda v, t: torch.from_numpy(np.concatenate(v) if isinstance(v, tuple) else np.asarray(v)).to(t).cuda()  # noqa: E731
    return {"tables": to(tables, I32), "free": to(free, I32), "count": to([len(stack)], I32), "lengths": to(after, I32),
            "starts": to(starts, I32), "slots": to((*slots, rest), I64), "positions": to((*positions, rest), I32),
            "requests": to((*requests, rest), I32)}


def _exact_turn(x, s):
    """The rotation as a product of complex numbers."""
    y, half = x.to(F64).clone(), s["freqs"].numel()
    one = torch.polar(torch.ones(1, dtype=F64, device="cuda"), torch.outer(s["positions"].to(F64), s["freqs"].to(F64)))
    if s["case"]["pairs"]:
        y[..., :2 * half] = torch.view_as_real(torch.view_as_complex(y[..., :2 * half].unflatten(-1, (half, 2)).contiguous())
                                               * one[:, None]).flatten(-2)
        return y
    z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * one[:, None]
    y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _exact_store(s):
    case = s["case"]
    page, result = case["page"], {"q": _exact_turn(s["q"], s)}
    for name, cache, y in (("k", s["kc"], _exact_turn(s["k"], s)), ("v", s["vc"], s["v"].to(F64))):
        c = _values(cache, case).to(F64)
        if case["type"] == "Q8_0":
            b = y.to(F32).to(F64).reshape(-1, 32)
            d = (b.abs().amax(1, keepdim=True) / 127).to(F32).to(F64)
            v = (b * torch.where(d > 0, (1 / d).to(F32).to(F64), 0.0)).to(F32).to(F64)
            # |v| <= 127, so every v and v + 1/2 is exact here
            y = (v.sign() * (v.abs() + 0.5).floor().clamp(max=127) * d.to(torch.float16).to(F64)).reshape(y.shape)
        c[s["slots"] // page, :, s["slots"] % page] = y
        result[name] = c
    return result


def _exact_attn(s):
    case = s["case"]
    H, K, D, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    out = s["out"].to(F64)
    for i, (r, last) in enumerate(zip(s["requests"].tolist(), s["positions"].tolist())):
        if r < 0:
            continue
        first = max(0, last + 1 - case["window"]) if case["window"] else 0
        pages = s["tables"][r, first // page:last // page + 1].long()
        k, v = (_values(c[pages], case).to(F64).transpose(0, 1).flatten(1, 2)[:, first % page:first % page + last + 1 - first]
                for c in (s["kc"], s["vc"]))
        z = (s["q"][i].to(F64).view(K, H // K, 1, D) * k[:, None]).sum(-1) / D ** 0.5
        out[i] = (torch.softmax(z, -1).unsqueeze(-1) * v[:, None]).sum(2).reshape(H, D) if last >= 0 else 0.0
    return out


def _exact_select(s):
    G, B, V = s["logits"].shape
    best = s["case"]["best"]
    scores, places = [], []
    for g in range(G):
        total = (torch.log_softmax(s["logits"][g].to(F64), -1) + s["scores"][g].to(F64)[:, None]).view(-1)
        for _ in range(best):  # the best one left, the lowest index of equal ones
            top = total.amax()
            at = (total == top).to(torch.uint8).argmax()
            scores.append(top)
            places.append(torch.where(top > NONE, at, -1))
            total[at] = NONE
    at = torch.stack(places).view(G, best)
    return {"scores": torch.stack(scores).view(G, best), "parents": torch.where(at < 0, -1, at // V).to(I32),
            "tokens": torch.where(at < 0, -1, at % V).to(I32)}


def _exact_reorder(s):
    case = s["case"]
    B, page = case["beams"], case["page"]
    tail, n = case["length"] // page, case["length"] % page
    old, kv = s["tables"].cpu(), _values(s["kv"], case).to(F64)
    tables, before = old.clone(), kv.clone()
    for i, p in enumerate(s["parents"].view(-1).tolist()):
        if p >= 0:
            parent = i - i % B + p
            tables[i, :tail] = old[parent, :tail]
            kv[:, int(old[i, tail]), :, :n] = before[:, int(old[parent, tail]), :, :n]
    return {"tables": tables.cuda(), "kv": kv}


EXACT = {"pages": _exact_pages, "store": _exact_store, "attn": _exact_attn, "select": _exact_select,
         "reorder": _exact_reorder}


def exact(case, seed):
    s = _inputs(case, seed)
    return EXACT[case["kind"]](s)
