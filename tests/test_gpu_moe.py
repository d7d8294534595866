"""rlq_moe_route and rlq_moe_ffn against plain implementations in 64 bits.

Tolerances.  The kernels add in f64 (n terms: off by at most n 2^-53 of the sum of
their magnitudes, below 2^-38 of it here) and round once to f32 (2^-24 of the
value), so a result is within 2^-24 |y| + 2^-38 sum|term| of the 64-bit one; a
further 2^-24 |w| covers a router weight that enters a product as f32.
The hidden values h are rounded to f32 and then to 8-bit levels by both sides from
f64 sums that agree to 2^-38: on these fixed inputs they round alike (checked by the
tolerance itself, which one differing level would break)."""
import numpy as np
import pytest

import oracle as O
from rlq_loader import load
from test_gpu_sweep import _weights

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType
TYPES = (DT.Q8_0, DT.Q2_K, DT.Q3_K, DT.Q4_K, DT.Q5_K, DT.Q6_K)


def say(*a):
    print("[case]", *a, flush=True)


@pytest.fixture(scope="module")
def ctx():
    c = rlq.Context(0)
    yield c
    c.close()


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


# ---- router ---------------------------------------------------------------------

def plain_route(router, x, k, gating="softmax", normalize=True, scale=1.0, bias=None):
    z = (x.astype(np.float64) @ router.astype(np.float64).T).astype(np.float32).astype(np.float64)
    if gating == "softmax":
        e = np.exp(z - z.max(1, keepdims=True))
        score = e / e.sum(1, keepdims=True)
    else:
        with np.errstate(over="ignore"):
            score = 1.0 / (1.0 + np.exp(-z))
    rank = z.copy() if bias is None else score + bias.astype(np.float64)
    rank[np.isnan(rank)] = -np.inf
    order = np.argsort(-rank, axis=1, kind="stable")[:, :k]
    none = np.take_along_axis(rank, order, 1) == -np.inf
    w = np.where(none, 0.0, np.take_along_axis(score, order, 1))
    if normalize:
        s = w.sum(1, keepdims=True)
        w = np.divide(w, s, out=np.zeros_like(w), where=s > 0)
    return z, np.where(none, -1, order).astype(np.int32), w * np.float64(np.float32(scale))


def check_route(ctx, router, x, k, **kw):
    bias = kw.get("bias")
    ids, w, z = ctx.moe_route(gpu(router), gpu(x), k, logits=True, **dict(kw, bias=None if bias is None else gpu(bias)))
    ids2, w2, none = ctx.moe_route(gpu(router), gpu(x), k, **dict(kw, bias=None if bias is None else gpu(bias)))
    ctx.sync()
    assert none is None and torch.equal(ids, ids2) and torch.equal(w, w2)
    wz, wi, ww = plain_route(router, x, k, **kw)
    size = np.abs(x.astype(np.float64)) @ np.abs(router.astype(np.float64)).T
    assert np.all(np.abs(z.cpu().numpy() - wz) <= 2.0 ** -23 * np.abs(wz) + 2.0 ** -38 * size)
    assert np.array_equal(ids.cpu().numpy(), wi)
    # f64 exponentials to a few units in the last place, a sum and a division, then one rounding to f32
    assert np.all(np.abs(w.cpu().numpy() - ww) <= (2.0 ** -24 + 2.0 ** -45) * np.abs(ww) + 2.0 ** -150)
    return ids, w


@pytest.mark.parametrize("tokens,experts,cols,k", [
    (1, 1, 1, 1), (1, 8, 4096, 2), (2, 2, 3, 2), (3, 16, 32, 4), (16, 17, 33, 5), (17, 8, 100, 8), (5, 64, 896, 6),
    (33, 65, 256, 7), (2, 128, 2048, 8), (70, 60, 224, 4), (4, 256, 512, 64), (3, 257, 96, 33), (2, 1024, 64, 64),
    (130, 1000, 36, 9), (1, 40, 30000, 3)])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_route(ctx, tokens, experts, cols, k, gating, normalize):
    say("route", tokens, experts, cols, k, gating, normalize)
    router, x = normal(1, experts, cols) * np.float32(1.5 / np.sqrt(cols)), normal(2, tokens, cols)
    check_route(ctx, router, x, k, gating=gating, normalize=normalize, scale=1.0 if normalize else 2.5)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_route_bias(ctx, gating):
    """The bias moves the choice, not the weights; -inf and NaN switch off."""
    say("route bias", gating)
    router, x = normal(3, 60, 128) * np.float32(0.1), normal(4, 21, 128)
    bias = normal(5, 60) * np.float32(0.3)
    bias[[0, 7, 59]] = -np.inf
    bias[13] = np.nan
    ids, _ = check_route(ctx, router, x, 6, gating=gating, bias=bias)
    assert not bool(torch.isin(ids, torch.tensor([0, 7, 13, 59], device="cuda", dtype=torch.int32)).any())
    bias[20] = np.inf
    ids, _ = check_route(ctx, router, x, 6, gating=gating, bias=bias)
    assert bool((ids[:, 0] == 20).all())


def test_route_with_too_few_experts(ctx):
    say("route few")
    router, x = normal(6, 9, 64), normal(7, 5, 64)
    bias = np.full(9, -np.inf, np.float32)
    ids, w = check_route(ctx, router, x, 4, bias=bias)  # none at all
    assert bool((ids == -1).all()) and bool((w == 0).all())
    bias[[2, 5]] = 0.0
    ids, w = check_route(ctx, router, x, 4, bias=bias)
    assert bool((ids[:, 2:] == -1).all()) and bool((ids[:, :2] >= 0).all())


def test_route_ties_go_to_the_lowest_index(ctx):
    say("route ties")
    row = normal(8, 1, 96)
    router = np.repeat(row, 130, axis=0)
    router[100] = 0.0
    ids, _ = check_route(ctx, router, normal(9, 4, 96), 8)
    assert bool((ids[0] == torch.arange(8, device="cuda")).all()) or int(ids[0, 0]) == 100
    check_route(ctx, np.zeros((70, 32), np.float32), normal(10, 2, 32), 5, bias=np.zeros(70, np.float32))


def test_route_of_extreme_logits(ctx):
    """Scores that underflow, and a saturated sigmoid."""
    say("route extreme")
    router, x = np.zeros((6, 4), np.float32), np.ones((2, 4), np.float32)
    router[:, 0] = [-2000.0, -1500.0, -900.0, -800.0, -760.0, -1000.0]
    for gating in ("softmax", "sigmoid"):
        for normalize in (True, False):
            check_route(ctx, router, x, 3, gating=gating, normalize=normalize)
    check_route(ctx, -router, x, 3, gating="sigmoid")


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_route_of_a_bad_token(ctx, bad):
    say("route bad", bad)
    router, x = normal(11, 20, 64), normal(12, 5, 64)
    x[3, 17] = bad
    ids, w, _ = ctx.moe_route(gpu(router), gpu(x), 3)
    with pytest.raises(rlq.QuantError) as e:
        ctx.sync()
    assert (e.value.name, e.value.a, e.value.b) == ("NonFinite", 4, 3)
    assert bool((ids[3] == -1).all()) and bool((w[3] == 0).all())
    keep = [0, 1, 2, 4]
    _, wi, _ = plain_route(router, x[keep], 3)
    assert np.array_equal(ids.cpu().numpy()[keep], wi)


def test_route_unaligned_and_refused(ctx):
    say("route unaligned")
    router, x = normal(13, 11, 64), normal(14, 3, 64)
    rs = torch.zeros(11 * 64 + 1, device="cuda")[1:].view(11, 64)
    rs.copy_(gpu(router))
    ids, w, _ = ctx.moe_route(rs, gpu(x), 2)
    _, wi, ww = plain_route(router, x, 2)
    assert np.array_equal(ids.cpu().numpy(), wi)
    with pytest.raises(ValueError):
        ctx.moe_route(gpu(router), gpu(x), 2, gating="tanh")
    with pytest.raises(ValueError):
        ctx.moe_route(gpu(router), gpu(x), 2, bias=gpu(normal(1, 10)))
    with pytest.raises(ValueError):
        ctx.moe_route(gpu(router), gpu(x), 2, ids=torch.zeros((3, 3), dtype=torch.int32, device="cuda"))
    with pytest.raises(rlq.QuantError) as e:
        ctx.moe_route(gpu(router), gpu(x), 12)
    assert e.value.name == "Shape"
    ids, w, _ = ctx.moe_route(gpu(router), gpu(x)[:0], 2)
    assert ids.shape == (0, 2)


# ---- experts ---------------------------------------------------------------------

def act(t):
    return DT.Q8_0 if t == DT.Q8_0 else DT.Q8_K


def unpacked(at, b, cols):
    """The numbers of packed activation rows, in 64 bits."""
    n, bs = O.row_bytes(int(at), cols), 32 if at == DT.Q8_0 else 256
    blocks = np.ascontiguousarray(b).reshape(-1, cols // bs, n * bs // cols)
    if at == DT.Q8_0:
        d, q = blocks[..., :2].copy().view(np.float16), blocks[..., 2:]
    else:
        d, q = blocks[..., :4].copy().view(np.float32), blocks[..., 4:260]
    return (d.astype(np.float64) * q.copy().view(np.int8)).reshape(-1, cols)


def quantized(at, x):
    x = np.ascontiguousarray(x, np.float32)
    return unpacked(at, np.concatenate([O.quantize(int(at), r) for r in x]), x.shape[1])


def values(t, data, rows, cols):
    """The weights' numbers in 64 bits: a level times a scale, less a minimum, from
    f16 scales and whole numbers.  The decoder's f32 products of those round, so the
    two parts are taken from decoded blocks with one of the scales cleared."""
    size = O.TYPE_SIZE[int(t)]
    b = np.frombuffer(bytes(data), np.uint8).reshape(-1, size).copy()
    halves = {DT.Q8_0: (0,), DT.Q2_K: (80, 82), DT.Q3_K: (108,), DT.Q4_K: (0, 2), DT.Q5_K: (0, 2), DT.Q6_K: (208,)}[t]
    out = 0.0
    for at in halves:
        one = b.copy()
        for o in halves:  # this scale 1, the others 0: whole numbers, exact in f32
            one[:, o:o + 2] = np.array([1.0 if o == at else 0.0], np.float16).view(np.uint8)
        whole = O.dequantize(int(t), one.reshape(-1), rows * cols).astype(np.float64).reshape(b.shape[0], -1)
        out = out + whole * b[:, at:at + 2].copy().view(np.float16).astype(np.float64)
    return out.reshape(rows, cols)


class Layer:
    def __init__(self, ctx, experts, cols, ffn, out, gate, down, seed=1):
        self.ctx, self.experts, self.cols, self.ffn, self.out, self.tg, self.td = ctx, experts, cols, ffn, out, gate, down
        shapes = ((gate, ffn, cols), (gate, ffn, cols), (down, out, ffn))
        data = [_weights(t, experts * r, c, seed + k) for k, (t, r, c) in enumerate(shapes)]
        self.w = [rlq.Weights(ctx, t, d, r, c, experts) for d, (t, r, c) in zip(data, shapes)]
        self.v = [values(t, d, experts * r, c).reshape(experts, r, c) for d, (t, r, c) in zip(data, shapes)]
        # weights of a size at which h is about 1
        self.size = float(np.sqrt(np.mean(self.v[0] ** 2) * cols))

    def x(self, seed, tokens):
        return normal(seed, tokens, self.cols) / np.float32(self.size)

    def call(self, x, ids, weights, **kw):
        return self.ctx.moe_ffn(*self.w, x, gpu(ids.astype(np.int32)), gpu(weights), **kw)

    def plain(self, a, ids, weights, residual=None):
        """(y, sum of the magnitudes of its terms) of numbers a, in 64 bits."""
        y = np.zeros((ids.shape[0], self.out)) if residual is None else residual.astype(np.float64)
        size = np.abs(y)
        for t in range(ids.shape[0]):
            for s in range(ids.shape[1]):
                e = ids[t, s]
                if e < 0:
                    continue
                g, u = ((self.v[k][e] @ a[t]).astype(np.float32).astype(np.float64) for k in (0, 1))
                with np.errstate(over="ignore"):
                    h = (g / (1 + np.exp(-g)) * u).astype(np.float32)
                q = quantized(act(self.td), h[None])[0]
                y = y.copy()
                y[t] += float(weights[t, s]) * (self.v[2][e] @ q)
                size[t] += abs(float(weights[t, s])) * (np.abs(self.v[2][e]) @ np.abs(q))
        return y, size

    def check(self, got, a, ids, weights, residual=None, rows=None):
        want, size = self.plain(a, ids, weights, residual)
        got = got.cpu().numpy().astype(np.float64)
        rows = range(ids.shape[0]) if rows is None else rows
        for t in rows:
            assert np.all(np.abs(got[t] - want[t]) <= 2.0 ** -24 * np.abs(want[t]) + 2.0 ** -38 * size[t]), t

    def close(self):
        for w in self.w:
            w.close()


def places(seed, tokens, experts, slots, dropped=0.0, twice=False):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(experts)[:slots] if slots <= experts else rng.integers(0, experts, slots)
                    for _ in range(tokens)]).astype(np.int32)
    if twice:
        ids[:, -1] = ids[:, 0]
    ids[rng.random(ids.shape) < dropped] = -1
    return ids, rng.random(ids.shape).astype(np.float32)


@pytest.mark.parametrize("tokens", [1, 2, 5, 8, 9, 16, 17, 32, 33])
@pytest.mark.parametrize("k", range(6))
def test_ffn_types(ctx, k, tokens):
    gate, down = TYPES[k], TYPES[(k + 2) % 6]
    say("ffn", gate.name, down.name, tokens)
    L = Layer(ctx, 5, 512, 768, 96, gate, down, 10 + k)
    ids, weights = places(20 + tokens, tokens, 5, 2, 0.15)
    x, res = L.x(30 + tokens, tokens), normal(31, tokens, 96)
    y = L.call(gpu(x), ids, weights, residual=gpu(res))
    ctx.sync()
    L.check(y, quantized(act(gate), x), ids, weights, res)
    L.close()


@pytest.mark.parametrize("gate,down,cols,ffn,out", [
    (DT.Q8_0, DT.Q8_0, 32, 32, 1), (DT.Q8_0, DT.Q8_0, 96, 288, 17), (DT.Q8_0, DT.Q4_K, 928, 256, 33),
    (DT.Q4_K, DT.Q8_0, 256, 1952, 100), (DT.Q6_K, DT.Q3_K, 4352, 256, 16), (DT.Q5_K, DT.Q2_K, 256, 4864, 15),
    (DT.Q3_K, DT.Q8_0, 2304, 64, 48), (DT.Q2_K, DT.Q6_K, 768, 2560, 31), (DT.Q8_0, DT.Q5_K, 4896, 512, 5)])
@pytest.mark.parametrize("tokens", [1, 6, 20])
def test_ffn_odd_sizes(ctx, gate, down, cols, ffn, out, tokens):
    """Rows of one block and of more blocks than waves, part chunks, part tiles."""
    say("ffn odd", gate.name, down.name, cols, ffn, out, tokens)
    L = Layer(ctx, 3, cols, ffn, out, gate, down, 40)
    ids, weights = places(41, tokens, 3, 2)
    x = L.x(42, tokens)
    y = L.call(gpu(x), ids, weights)
    ctx.sync()
    L.check(y, quantized(act(gate), x), ids, weights)
    L.close()


@pytest.mark.parametrize("gate", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("tokens", [1, 7, 18])
def test_ffn_packed(ctx, gate, tokens):
    say("ffn packed", gate.name, tokens)
    L = Layer(ctx, 6, 768, 512, 64, gate, DT.Q4_K, 50)
    ids, weights = places(51, tokens, 6, 3)
    at = act(gate)
    q = ctx.quantize(at, gpu(L.x(52, tokens))).view(tokens, -1)
    y = L.call(q, ids, weights, x_dtype=at)
    ctx.sync()
    L.check(y, unpacked(at, q.cpu().numpy(), 768), ids, weights)
    L.close()


def test_ffn_packed_extremes(ctx):
    """Levels of -128, scales of 0, and bsums that do not belong to the levels."""
    say("ffn packed extremes")
    for gate in (DT.Q4_K, DT.Q2_K, DT.Q6_K):
        L = Layer(ctx, 2, 512, 256, 32, gate, DT.Q4_K, 55)
        rng = np.random.default_rng(56)
        b = np.zeros((3, 2, 292), np.uint8)
        b[..., :4] = np.array([1e-3], np.float32).view(np.uint8)
        b[..., 4:260] = rng.integers(0, 256, (3, 2, 256), dtype=np.uint8)
        b[0, 0, 4:260] = 128
        b[1, 1, :4] = 0
        b[..., 260:] = 0x7f  # not looked at
        ids, weights = places(57, 3, 2, 1)
        y = L.call(gpu(b.reshape(3, -1)), ids, weights, x_dtype=DT.Q8_K)
        ctx.sync()
        L.check(y, unpacked(DT.Q8_K, b, 512), ids, weights)
        L.close()


def test_ffn_of_many_experts_and_places(ctx):
    """More experts than waves of the plan, all places of a token, every token the
    same expert, one token alone with an expert."""
    say("ffn many")
    L = Layer(ctx, 700, 256, 32, 16, DT.Q8_0, DT.Q8_0, 60)
    ids, weights = places(61, 32, 700, 64)
    x = L.x(62, 32)
    y = L.call(gpu(x), ids, weights)
    ctx.sync()
    L.check(y, quantized(DT.Q8_0, x), ids, weights)
    for ids in (np.full((40, 1), 699), np.full((31, 2), 3), np.array([[i, 699 - i] for i in range(9)])):
        weights = np.random.default_rng(63).random(ids.shape).astype(np.float32)
        x = L.x(64, len(ids))
        y = L.call(gpu(x), ids, weights)
        ctx.sync()
        L.check(y, quantized(DT.Q8_0, x), ids, weights)
    L.close()


@pytest.mark.parametrize("tokens", [1, 4, 12, 25])
def test_ffn_of_no_expert_and_of_one_twice(ctx, tokens):
    """Places of -1 (whatever their weight), tokens without any, and an expert that
    a token names twice."""
    say("ffn none", tokens)
    L = Layer(ctx, 4, 512, 512, 40, DT.Q4_K, DT.Q6_K, 70)
    x, res = L.x(71, tokens), normal(72, tokens, 40)
    ids, weights = places(73, tokens, 4, 3, 0.0, True)
    ids[0] = -1
    weights[0] = np.nan
    ids[-1, 1] = -1
    weights[-1, 1] = np.inf
    y = L.call(gpu(x), ids, weights, residual=gpu(res))
    ctx.sync()
    assert np.array_equal(y[0].cpu().numpy(), res[0])
    L.check(y, quantized(DT.Q8_K, x), ids, np.where(ids < 0, np.float32(0), weights), res)
    none = np.full_like(ids, -1)
    y = L.call(gpu(x), none, weights)
    ctx.sync()
    assert bool((y == 0).all())
    y = L.call(gpu(x), none, weights, residual=gpu(res))
    ctx.sync()
    assert np.array_equal(y.cpu().numpy(), res)
    L.close()


def test_ffn_weights_that_are_not_finite(ctx):
    """They pass into y of their own token only."""
    say("ffn weights")
    L = Layer(ctx, 3, 256, 256, 24, DT.Q5_K, DT.Q5_K, 75)
    ids, weights = places(76, 4, 3, 2)
    weights[1, 0], weights[2, 1] = np.nan, np.inf
    x = L.x(77, 4)
    y = L.call(gpu(x), ids, weights)
    ctx.sync()
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[2]).any())
    L.check(y, quantized(DT.Q8_K, x), ids, weights, rows=[0, 3])
    L.close()


@pytest.mark.parametrize("gate,down", [(DT.Q4_K, DT.Q6_K), (DT.Q8_0, DT.Q8_0), (DT.Q2_K, DT.Q3_K), (DT.Q5_K, DT.Q4_K)])
def test_ffn_does_not_depend_on_company(ctx, gate, down):
    """A token's row has the same bits alone, in a batch, and past 32 tokens."""
    say("ffn company", gate.name, down.name)
    L = Layer(ctx, 8, 1024, 1536, 128, gate, down, 80)
    tokens = 37
    ids, weights = places(81, tokens, 8, 2)
    x, res = L.x(82, tokens), normal(83, tokens, 128)
    y = L.call(gpu(x), ids, weights, residual=gpu(res))
    for cut in (slice(0, 1), slice(5, 12), slice(3, 16), slice(10, 37), slice(36, 37)):
        part = L.call(gpu(x[cut]), ids[cut], weights[cut], residual=gpu(res[cut]))
        assert torch.equal(part, y[cut]), cut
    ctx.sync()
    L.close()


def test_ffn_in_place_and_on_other_streams(ctx):
    say("ffn streams")
    L = Layer(ctx, 6, 512, 512, 512, DT.Q4_K, DT.Q4_K, 90)
    ids, weights = places(91, 5, 6, 2)
    x, res = L.x(92, 5), normal(93, 5, 512)
    want = L.call(gpu(x), ids, weights, residual=gpu(res))
    h = gpu(res)
    assert L.call(gpu(x), ids, weights, residual=h, y=h) is h
    assert torch.equal(h, want)
    ctx.sync()
    other, s = rlq.Context(0), torch.cuda.Stream()  # two contexts, two streams at once
    args = gpu(x), gpu(ids), gpu(weights)
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        outs.append(ctx.moe_ffn(*L.w, args[0], args[1], args[2]))
        with torch.cuda.stream(s):
            outs.append(other.moe_ffn(*L.w, args[0], args[1], args[2]))
    ctx.sync(), other.sync(s)
    want = ctx.moe_ffn(*L.w, *args)
    assert all(torch.equal(o, want) for o in outs)
    ctx.sync()
    other.close()
    L.close()


@pytest.mark.parametrize("tokens", [1, 3, 33])
@pytest.mark.parametrize("what", ["id high", "id low", "nan", "inf", "tiny", "h inf", "h tiny"])
def test_ffn_of_a_bad_token(ctx, what, tokens):
    """Its row of y stays as it was, the others are written."""
    say("ffn bad", what, tokens)
    L = Layer(ctx, 4, 512, 512, 48, DT.Q4_K, DT.Q6_K, 100)
    ids, weights = places(101, tokens, 4, 2)
    x, bad = L.x(102, tokens), tokens - 1
    name, a, b = "NonFinite", 3, bad
    if what == "id high":
        ids[bad, 1], name, a, b = 4, "Bounds", bad * 2 + 1, 0
    elif what == "id low":
        ids[bad, 0], name, a, b = -2, "Bounds", bad * 2, 0
    elif what == "nan":
        x[bad, 300], name, a = np.nan, "NonFiniteInput", 300
    elif what == "inf":
        x[bad, 511], name, a = -np.inf, "NonFiniteInput", 511
    elif what == "tiny":  # the first block's scale is not finite
        x[bad, :256], name, a = 1e-38, "UnrepresentableScale", 0
    elif what == "h inf":  # g u past the largest f32
        x[bad] *= np.float32(1e25)
    else:  # h of 1e-38 and less, not 0
        x[bad] *= np.float32(1e-19)
        name, a = "UnrepresentableScale", 0
    y = torch.full((tokens, 48), 7.0, device="cuda")
    L.call(gpu(x), ids, weights, y=y)
    with pytest.raises(rlq.QuantError) as e:
        ctx.sync()
    assert (e.value.name, e.value.a, e.value.b) == (name, a, b)
    assert bool((y[bad] == 7.0).all())
    good = [t for t in range(tokens) if t != bad]
    L.check(y, quantized(DT.Q8_K, np.where(np.arange(tokens)[:, None] == bad, np.float32(0), x)), np.where(
        np.arange(tokens)[:, None] == bad, -1, ids), weights, rows=good)
    ctx.sync()  # cleared, and the next call is whole
    x, (ids, weights) = L.x(103, tokens), places(104, tokens, 4, 2)
    L.call(gpu(x), ids, weights, y=y)
    ctx.sync()
    L.check(y, quantized(DT.Q8_K, x), ids, weights)
    L.close()


def test_ffn_shapes_refused(ctx):
    L = Layer(ctx, 2, 256, 256, 16, DT.Q4_K, DT.Q4_K, 110)
    ids, weights = places(111, 3, 2, 1)
    x = gpu(L.x(112, 3))
    for kw in (dict(y=torch.zeros((2, 16), device="cuda")), dict(residual=torch.zeros(16, device="cuda"))):
        with pytest.raises(ValueError):
            L.call(x, ids, weights, **kw)
    with pytest.raises(ValueError):
        L.call(x[:2], ids, weights)
    with pytest.raises(ValueError):
        L.call(x, ids, weights[:2])
    with pytest.raises(TypeError):
        L.call(x.double(), ids, weights)
    with pytest.raises(rlq.QuantError) as e:
        L.call(torch.zeros((3, 272), dtype=torch.uint8, device="cuda"), ids, weights, x_dtype=DT.Q8_0)
    assert e.value.name == "Unsupported"
    assert L.call(x[:0], ids[:0], weights[:0]).shape == (0, 16)
    ctx.sync()
    L.close()


def test_replayed_layer(ctx):
    """Norm, router and experts as one recorded sequence, its scratch outliving the
    growth that larger calls between the replays bring."""
    say("layer replayed")
    c = rlq.Context(0)
    L = Layer(c, 8, 512, 1024, 512, DT.Q4_K, DT.Q6_K, 120)
    big = Layer(c, 16, 512, 512, 256, DT.Q8_0, DT.Q8_0, 121)
    router, norm = gpu(normal(122, 8, 512) * np.float32(0.05)), gpu(1 + normal(123, 512) * np.float32(0.05))
    att, hidden = torch.zeros((4, 512), device="cuda"), torch.zeros((4, 512), device="cuda")
    out = torch.zeros((4, 512), device="cuda")

    def layer(att, hidden, out):
        total, y, q = c.rms_norm(att, norm, 1e-5, residual=hidden, packed=DT.Q8_K)
        ids, weights, _ = c.moe_route(router, y, 2)
        return c.moe_ffn(*L.w, q, ids, weights, x_dtype=DT.Q8_K, residual=total, y=out)

    layer(att, hidden, out)
    c.sync()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        layer(att, hidden, out)
    fill = []
    for k in range(4):
        att.copy_(gpu(normal(130 + k, 4, 512))), hidden.copy_(gpu(normal(140 + k, 4, 512)))
        out.zero_()
        graph.replay()
        got = out.clone()
        want = layer(att, hidden, torch.empty_like(out))
        c.sync()
        assert torch.equal(got, want) and bool(torch.isfinite(got).all())
        n = 8 * (k + 1)
        ids, weights = places(150, n, 16, 4)
        big.call(gpu(big.x(151, n)), ids, weights)
        c.moe_route(gpu(normal(152, 64, 64)), gpu(normal(153, 100 * n, 64)), 2)
        c.sync()
        fill += [torch.full((m,), 1e30, device="cuda") for m in (1 << 10, 1 << 14, 1 << 18, 1 << 20)]
    L.close(), big.close(), c.close()


@pytest.mark.parametrize("tokens", [1, 6])
def test_layer_of_the_three(ctx, tokens):
    """A decoder layer's second half, from the residual stream to the next one,
    against 64 bits; and the experts' products against mul_mat_id's own."""
    say("layer", tokens)
    L = Layer(ctx, 8, 1024, 1280, 1024, DT.Q4_K, DT.Q6_K, 160)
    router, norm = normal(161, 8, 1024) * np.float32(0.04), 1 + normal(162, 1024) * np.float32(0.05)
    att, hidden = normal(163, tokens, 1024), normal(164, tokens, 1024)
    total, y, q = ctx.rms_norm(gpu(att), gpu(norm.astype(np.float32)), 1e-5, residual=gpu(hidden), packed=DT.Q8_K)
    ids, weights, _ = ctx.moe_route(gpu(router), y, 2)
    out = ctx.moe_ffn(*L.w, q, ids, weights, x_dtype=DT.Q8_K, residual=total)
    ctx.sync()
    t = att + hidden
    normed = np.stack([O.rms_norm(r, norm.astype(np.float32), 1e-5) for r in t])
    _, wi, ww = plain_route(router, normed, 2)
    assert np.array_equal(ids.cpu().numpy(), wi)
    L.check(out, quantized(DT.Q8_K, normed), wi, weights.cpu().numpy(), t)
    # g and u as mul_mat_id has them, in its f32 order: within the 1e-5 of its batched products
    g = ctx.mul_mat_id(L.w[0], y.view(tokens, 1, -1), ids).cpu().numpy()
    a = quantized(DT.Q8_K, normed)
    want = np.stack([[L.v[0][e] @ a[k] for e in wi[k]] for k in range(tokens)])
    assert np.linalg.norm(g - want) <= 1e-5 * np.linalg.norm(want)
    ctx.sync()
    L.close()


@pytest.mark.parametrize("slots,cols,ffn,out,gate,down", [
    (63, 256, 1024, 2080, DT.Q8_0, DT.Q8_0), (64, 256, 1024, 2080, DT.Q8_0, DT.Q8_0),
    (63, 256, 1024, 2080, DT.Q4_K, DT.Q5_K), (64, 256, 1024, 2080, DT.Q4_K, DT.Q2_K),
    (3, 32768, 64, 16, DT.Q8_0, DT.Q8_0), (3, 32800, 64, 16, DT.Q8_0, DT.Q8_0),
    (2, 32768, 256, 40, DT.Q4_K, DT.Q6_K), (2, 33024, 256, 40, DT.Q5_K, DT.Q3_K)])
def test_ffn_of_one_token_at_its_limits(ctx, slots, cols, ffn, out, gate, down):
    """More places than experts, and as many values of x and of h as fit the LDS, and more."""
    say("ffn one", slots, cols, ffn, out, gate.name, down.name)
    L = Layer(ctx, 2, cols, ffn, out, gate, down, 170)
    ids, weights = places(171, 1, 2, slots)
    x = L.x(172, 1)
    y = L.call(gpu(x), ids, weights)
    ctx.sync()
    L.check(y, quantized(act(gate), x), ids, weights)
    L.close()


@pytest.mark.parametrize("tokens", [1, 3, 33])
def test_ffn_does_not_look_at_x_without_experts(ctx, tokens):
    say("ffn unseen x", tokens)
    L = Layer(ctx, 3, 512, 256, 48, DT.Q4_K, DT.Q4_K, 175)
    ids, weights = places(176, tokens, 3, 2)
    x, res = L.x(177, tokens), normal(178, tokens, 48)
    for t in {0, tokens - 1}:
        ids[t] = -1
        x[t, 5], x[t, 400] = np.nan, np.inf
    y = L.call(gpu(x), ids, weights, residual=gpu(res))
    ctx.sync()
    L.check(y, quantized(DT.Q8_K, np.where((ids < 0).all(1, keepdims=True), np.float32(0), x)), ids, weights, res)
    L.close()


@pytest.mark.parametrize("down", [DT.Q4_K, DT.Q8_0], ids=lambda t: t.name)
@pytest.mark.parametrize("tokens", [8, 16, 32])
def test_ffn_of_several_bad_tokens(ctx, tokens, down):
    """Every way of a token to fail in one call, where workgroups share the tiles of y."""
    say("ffn several bad", tokens, down.name)
    L = Layer(ctx, 4, 512, 4096, 48, DT.Q4_K, down, 180)
    ids, weights = places(181, tokens, 4, 2)
    x, res = L.x(182, tokens), normal(183, tokens, 48)
    x[1, 300] = np.nan
    x[2] *= np.float32(1e25)   # h is infinite
    x[3] *= np.float32(1e-19)  # h's scale is (nearly) not a number
    weights[4, 0] = np.nan     # no error
    ids[5, 1] = 9
    y = torch.full((tokens, 48), 7.0, device="cuda")
    L.call(gpu(x), ids, weights, residual=gpu(res), y=y)
    with pytest.raises(rlq.QuantError) as e:
        ctx.sync()
    assert (e.value.name, e.value.a) == ("Bounds", 11)
    assert bool((y[[1, 2, 3, 5]] == 7.0).all()) and bool(torch.isnan(y[4]).all())
    good = [t for t in range(tokens) if t not in (1, 2, 3, 4, 5)]
    x[1:6], ids[1:6] = 0, -1
    L.check(y, quantized(DT.Q8_K, x), ids, weights, res, rows=good)
    ctx.sync()
    L.close()


@pytest.mark.parametrize("tokens,experts,cols,k", [(1, 8, 1024, 2), (3, 128, 512, 8), (40, 128, 2048, 8), (300, 60, 896, 6),
                                                   (20, 30, 17000, 3)])
def test_route_replayed(ctx, tokens, experts, cols, k):
    """The counts by which workgroups know each other are as they were after every
    call: replays among eager calls of other sizes."""
    say("route replayed", tokens, experts, cols, k)
    c = rlq.Context(0)
    router, x = gpu(normal(190, experts, cols) / np.float32(np.sqrt(cols))), torch.zeros((tokens, cols), device="cuda")
    c.moe_route(router, x, k)
    c.sync()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ids, weights, _ = c.moe_route(router, x, k)
    for n in range(4):
        rows = normal(191 + n, tokens, cols)
        x.copy_(gpu(rows))
        graph.replay()
        wi, ww = plain_route(router.cpu().numpy(), rows, k)[1:]
        assert np.array_equal(ids.cpu().numpy(), wi)
        assert np.all(np.abs(weights.cpu().numpy() - ww) <= (2.0 ** -24 + 2.0 ** -45) * np.abs(ww) + 2.0 ** -150)
        eager = c.moe_route(router, x, k)
        assert torch.equal(eager[0], ids) and torch.equal(eager[1], weights)
        check_route(c, normal(195, 64, 64), normal(196 + n, 50 * n + 1, 64), 2)
    c.sync()
    c.close()


@pytest.mark.parametrize("tokens", [1, 7, 33])
def test_ffn_replayed(ctx, tokens):
    say("ffn replayed", tokens)
    c = rlq.Context(0)
    L = Layer(c, 6, 512, 2048, 256, DT.Q5_K, DT.Q6_K, 200)
    x, ids, weights = torch.zeros((tokens, 512), device="cuda"), *map(gpu, places(201, tokens, 6, 2))
    c.moe_ffn(*L.w, x, ids, weights)
    c.sync()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = c.moe_ffn(*L.w, x, ids, weights)
    for n in range(4):
        i, w = places(202 + n, tokens, 6, 2, 0.2)
        ids.copy_(gpu(i)), weights.copy_(gpu(w)), x.copy_(gpu(L.x(206 + n, tokens)))
        graph.replay()
        eager = c.moe_ffn(*L.w, x, ids, weights)
        c.sync()
        assert torch.equal(y, eager)
        L.check(y, quantized(DT.Q8_K, x.cpu().numpy()), i, w)
        other = 1 + 12 * n  # of another number of parts
        i, w = places(210, other, 6, 2)
        c.moe_ffn(*L.w, gpu(L.x(211, other)), gpu(i), gpu(w))
    c.sync()
    L.close(), c.close()


HALF = {DT.Q8_0: 0, DT.Q2_K: 80, DT.Q3_K: 108, DT.Q4_K: 0, DT.Q5_K: 2, DT.Q6_K: 208}  # a scale (Q5_K: the minimums') in a block


@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("tokens", [1, 2, 7, 14, 30])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_ffn_of_an_expert_with_a_bad_scale(ctx, t, tokens, bad):
    """One scale of one row of an expert: the tokens that use it see it in that row of y
    (of gate: they have no h), the others have the bits of a sound expert."""
    say("ffn bad scale", t.name, tokens, bad)
    E, K, F, R, size, rb = 4, 512, 2048, 40, O.TYPE_SIZE[int(t)], 32 if t == DT.Q8_0 else 256
    gate, up, down = (_weights(t, E * r, c, 220 + k) for k, (r, c) in enumerate(((F, K), (F, K), (R, F))))

    def weights(data, rows, cols, hurt):
        b = np.frombuffer(bytes(data), np.uint8).copy().reshape(E, rows, cols // rb, size)
        if hurt:
            b[2, 7, -1, HALF[t]:HALF[t] + 2] = np.array([bad], np.float16).view(np.uint8)
        return rlq.Weights(ctx, t, b.reshape(-1), rows, cols, E)

    clean = [weights(gate, F, K, False), weights(up, F, K, False), weights(down, R, F, False)]
    hurt = [weights(gate, F, K, True), weights(down, R, F, True)]
    ids, w = places(221, tokens, E, 2)
    ids[0] = [1, 2]
    mean = float(np.sqrt(np.mean(values(t, gate, E * F, K) ** 2) * K))
    x, ids_d, w_d = gpu(normal(222, tokens, K) / np.float32(mean)), gpu(ids), gpu(w)
    uses = torch.from_numpy((ids == 2).any(1)).cuda()
    want = ctx.moe_ffn(*clean, x, ids_d, w_d)
    ctx.sync()
    y = ctx.moe_ffn(clean[0], clean[1], hurt[1], x, ids_d, w_d)
    ctx.sync()
    assert torch.equal(y[~uses], want[~uses]) and not bool(torch.isfinite(y[uses][:, 7]).any())
    keep = [r for r in range(R) if r != 7]
    assert torch.equal(y[:, keep], want[:, keep])
    one = ctx.moe_ffn(clean[0], clean[1], hurt[1], x[:1].contiguous(), ids_d[:1].contiguous(), w_d[:1].contiguous())
    assert torch.equal(one.nan_to_num(nan=123.0), y[:1].nan_to_num(nan=123.0))
    ctx.sync()
    y = torch.full((tokens, R), 7.0, device="cuda")
    ctx.moe_ffn(hurt[0], clean[1], clean[2], x, ids_d, w_d, y=y)
    with pytest.raises(rlq.QuantError) as e:
        ctx.sync()
    assert (e.value.name, e.value.a, e.value.b) == ("NonFinite", 3, 0)
    assert torch.equal(y[~uses], want[~uses]) and bool((y[uses] == 7.0).all())
    for m in clean + hurt:
        m.close()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("packed", [False, True])
def test_ffn_of_one_token_with_many_tiles(ctx, t, packed):
    """Enough rows of h for K to be split less, and as many of K's chunks as waves, fewer and more."""
    say("ffn many tiles", t.name, packed)
    for cols in (256, 768):
        L = Layer(ctx, 2, cols, 2304, 48, t, DT.Q8_0, 230)
        ids, weights = places(231, 1, 2, 16)
        x = L.x(232, 1)
        if packed:
            q = ctx.quantize(act(t), gpu(x)).view(1, -1)
            y, a = L.call(q, ids, weights, x_dtype=act(t)), unpacked(act(t), q.cpu().numpy(), cols)
        else:
            y, a = L.call(gpu(x), ids, weights), quantized(act(t), x)
        ctx.sync()
        L.check(y, a, ids, weights)
        L.close()


@pytest.mark.parametrize("t", [DT.Q8_0, DT.Q4_K], ids=lambda t: t.name)
def test_ffn_of_some_tokens_with_many_tiles(ctx, t):
    say("ffn many tiles, some tokens", t.name)
    L = Layer(ctx, 20, 512, 3584, 24, t, DT.Q6_K, 235)
    ids, weights = places(236, 13, 20, 4)
    x = L.x(237, 13)
    y = L.call(gpu(x), ids, weights)
    ctx.sync()
    L.check(y, quantized(act(t), x), ids, weights)
    L.close()


@pytest.mark.parametrize("tokens", [1, 4, 12, 25, 33])
def test_ffn_of_no_expert_keeps_the_residuals_bits(ctx, tokens):
    """A token without any expert gets its residual: -0 as -0."""
    say("ffn residual bits", tokens)
    L = Layer(ctx, 4, 256, 256, 40, DT.Q4_K, DT.Q6_K, 240)
    ids, weights = places(241, tokens, 4, 2)
    res = normal(242, tokens, 40)
    res[:, ::3] = -0.0
    for t in {0, tokens // 2, tokens - 1}:
        ids[t] = -1
    none = (ids < 0).all(1)
    x = L.x(243, tokens)
    y = L.call(gpu(x), ids, weights, residual=gpu(res))
    ctx.sync()
    assert np.array_equal(y.cpu().numpy().view(np.uint32)[none], res.view(np.uint32)[none])
    L.check(y, quantized(DT.Q8_K, x), ids, weights, res)
    y = gpu(res)
    L.call(gpu(x), np.full_like(ids, -1), weights, residual=y, y=y)
    ctx.sync()
    assert np.array_equal(y.cpu().numpy().view(np.uint32), res.view(np.uint32))
    y = L.call(gpu(x), np.full_like(ids, -1), weights)  # no residual: 0
    ctx.sync()
    assert not y.cpu().numpy().view(np.uint32).any()
    L.close()


@pytest.mark.parametrize("scale", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_route_scale_that_is_not_finite(ctx, gating, scale):
    """Places without an expert, and those of a normalized sum of 0, have weights of
    0 whatever the scale; the others are the scale's."""
    say("route scale", gating, scale)
    router, x = normal(250, 9, 64), normal(251, 5, 64)
    bias = np.full(9, -np.inf, np.float32)
    bias[[2, 5]] = 0.0
    for normalize in (True, False):
        ids, w, _ = ctx.moe_route(gpu(router), gpu(x), 4, gating=gating, normalize=normalize, scale=scale, bias=gpu(bias))
        ctx.sync()
        ids, w = ids.cpu().numpy(), w.cpu().numpy()
        assert (ids[:, :2] >= 0).all() and (ids[:, 2:] == -1).all()
        assert not w[:, 2:].view(np.uint32).any()
        assert np.isnan(w[:, :2]).all() if np.isnan(scale) else (w[:, :2] == scale).all()
    router, x = np.zeros((6, 4), np.float32), np.ones((2, 4), np.float32)
    router[:, 0] = -800.0  # sigmoids of 0
    _, w, _ = ctx.moe_route(gpu(router), gpu(x), 3, gating="sigmoid", scale=scale)
    ctx.sync()
    assert not w.cpu().numpy().view(np.uint32).any()


@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_ffn_with_many_tiles_in_any_company(ctx, t):
    """Experts of enough rows for K to be split less, from one token (two waves) to eight
    (four), sixteen and more (two): 64 bits for all tokens, and the same bits in all of
    these calls.  (Other orders of the f64 sums of n terms t round apart for at most
    n 2^-28 sum|t| / |sum| of the values.  Here y has 16 values a token, of 70 terms
    and a ratio near 8: about one call of 33 tokens in 1000 at the most.  Of g and u, n is
    2, and the one in 256 that is its block's largest moves y.)"""
    say("ffn many tiles, company", t.name)
    L = Layer(ctx, 19, 512, 3584, 16, t, DT.Q6_K, 270)
    ids, weights = places(271, 33, 19, 5, 0.05)
    x, res = L.x(272, 33), normal(273, 33, 16)
    y = L.call(gpu(x), ids, weights, residual=gpu(res))
    ctx.sync()
    L.check(y, quantized(act(t), x), ids, weights, res)
    for cut in (slice(0, 1), slice(7, 8), slice(1, 9), slice(3, 19), slice(20, 30), slice(14, 33)):
        part = L.call(gpu(x[cut]), ids[cut], weights[cut], residual=gpu(res[cut]))
        assert torch.equal(part, y[cut]), cut
    ctx.sync()
    L.close()


@pytest.mark.parametrize("tokens,experts,cols,k", [(3, 11, 64, 2), (2, 100, 4096, 5), (5, 300, 36, 9), (300, 128, 2048, 8),
                                                   (20, 30, 17000, 3), (33, 300, 16500, 4)])
@pytest.mark.parametrize("which", ["x", "router", "both"])
def test_route_of_unaligned_tensors(ctx, tokens, experts, cols, k, which):
    """Both kernels' loads of x and of the router without 16-byte alignment."""
    say("route unaligned", tokens, experts, cols, k, which)
    router, x = normal(280, experts, cols) * np.float32(1.5 / np.sqrt(cols)), normal(281, tokens, cols)

    def off(a):
        return torch.cat([torch.zeros(1, device="cuda"), gpu(a).view(-1)])[1:].view(a.shape)

    r, z = (off(router) if which != "x" else gpu(router)), (off(x) if which != "router" else gpu(x))
    ids, w, logits = ctx.moe_route(r, z, k, logits=True)
    aligned = ctx.moe_route(gpu(router), gpu(x), k, logits=True)
    ctx.sync()
    assert torch.equal(ids, aligned[0]) and torch.equal(w, aligned[1]) and torch.equal(logits, aligned[2])
    _, wi, ww = plain_route(router, x, k)
    assert np.array_equal(ids.cpu().numpy(), wi)
    assert np.all(np.abs(w.cpu().numpy() - ww) <= (2.0 ** -24 + 2.0 ** -45) * np.abs(ww) + 2.0 ** -150)
