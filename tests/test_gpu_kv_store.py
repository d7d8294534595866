"""rlq_kv_store: the place that an error names, within the four values of a thread too, slots named twice, and token sizes on
both sides of every border between its kernels."""
import numpy as np
import pytest

from rlq_loader import load
from test_gpu_kv import cuda, raises, say, store

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType


@pytest.fixture(scope="module")
def ctx():
    c = rlq.Context(0)
    yield c
    c.close()


def planted(ctx, dtype, half, pairs, at, value=np.nan, token=1):
    """Stores three tokens (heads 4 and 2 of 128), `value` at the places `at` in [q | k | v] of one of them."""
    rng = np.random.default_rng(half)
    x = rng.standard_normal((3, 8 * 128)).astype(np.float32)
    x[token, at] = value
    x = cuda(x).unflatten(1, (8, 128))
    cache = rlq.KvCache.make(dtype, 1, 2, 16, 128)
    freqs = cuda(np.full(half, 0.01, np.float32)) if half else None
    ctx.kv_store(cache, x[:, 4:6], x[:, 6:], cuda(np.arange(3)), x[:, :4], cuda(np.arange(3, dtype=np.int32)), freqs, pairs)


@pytest.mark.parametrize("half", [0, 32, 7])  # (7: no whole fours of rotated values)
@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_store_error_names_the_value(ctx, dtype, half):
    """NaN and what the cache's type does not hold, at every place of a four, in values that are not rotated."""
    for part in (0, 4 * 128, 6 * 128):
        for e in (100, 101, 102, 103, 127):
            say("store error place", dtype, half, part, e)
            planted(ctx, dtype, half, False, part + e)
            with raises("NonFiniteInput", part + e, 1):
                ctx.sync()
    large = {DT.F32: np.inf, DT.F16: -65520.0, DT.BF16: 3.4e38, DT.Q8_0: np.inf}[dtype]
    for places in ((6 * 128 + 103,), (4 * 128 + 67, 4 * 128 + 65, 6 * 128 + 3), (6 * 128 + 94, 6 * 128 + 95)):
        say("store error place", dtype, half, places)
        planted(ctx, dtype, half, False, list(places), large)
        with raises("NonFiniteInput", min(places), 1):
            ctx.sync()


@pytest.mark.parametrize("half,pairs", [(32, False), (32, True), (7, False), (7, True), (64, True), (64, False)])
def test_store_error_of_rotated_values(ctx, half, pairs):
    """Both values of a rotated pair are no numbers where one was none: the first of them is named."""
    for head in (0, 3, 4, 5):
        for i in (0, 1, 2, 3, half - 1):
            first, second = (2 * i, 2 * i + 1) if pairs else (i, i + half)
            for e in (first, second):
                say("store error pair", half, pairs, head, e)
                planted(ctx, DT.F16, half, pairs, head * 128 + e)
                with raises("NonFiniteInput", head * 128 + first, 1):
                    ctx.sync()


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_store_of_a_slot_named_twice(ctx, dtype):
    """What lies in a slot that several tokens name is each of them's in part: every value (of Q8_0 every level and every
    scale) is one of the tokens', and every other slot is as without them."""
    say("store slot twice", dtype)
    tokens, kv, dim = 600, 2, 128
    x = torch.arange(1, tokens + 1, device="cuda", dtype=torch.float32).view(-1, 1, 1).expand(tokens, kv, dim).contiguous() / 1024
    slots = torch.arange(tokens, device="cuda") % 7 + 16
    slots[50] = 3
    cache = rlq.KvCache.make(dtype, 3, kv, 16, dim)
    ctx.kv_store(cache, x, -x, slots)
    ctx.sync()
    alone = rlq.KvCache.make(dtype, 40, kv, 16, dim)
    ctx.kv_store(alone, x, -x, torch.arange(tokens, device="cuda"))
    ctx.sync()

    def parts(t):  # levels and scales, or values: [kv, tokens, ..]
        if dtype != DT.Q8_0:
            return [t.transpose(0, 1).reshape(kv, -1, dim)]
        levels, scales = t[..., :16 * dim], t[..., 16 * dim:].contiguous().view(torch.float16)
        return [levels.unflatten(-1, (16, dim)).transpose(0, 1).reshape(kv, -1, dim),
                scales.unflatten(-1, (16, dim // 32)).transpose(0, 1).reshape(kv, -1, dim // 32)]

    for t, own in ((cache.k, alone.k), (cache.v, alone.v)):
        for got, each in zip(parts(t), parts(own)):
            for s in range(48):
                named = [i for i in range(tokens) if int(slots[i]) == s] if s != 3 else [50]
                if not named:
                    assert (got[:, s] == 0).all()
                    continue
                assert (got[:, s].unsqueeze(1) == each[:, named]).any(1).all(), s


# Fours of values a token: to 512, 1024, 2048 and more of many tokens (more than CUs), to 1024, 2048, 4096 and more of few.
SIZES = [(12, 2, 128), (13, 2, 128), (7, 3, 160), (28, 2, 128), (29, 2, 128), (23, 1, 192), (48, 8, 128), (49, 8, 128), (64, 8, 128),
         (112, 8, 128), (113, 8, 128), (40, 4, 224), (0, 40, 128)]


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("heads,kv,dim", SIZES)
def test_store_sizes(ctx, dtype, heads, kv, dim):
    """Bit for bit, of few and of many tokens, into new queries and in place, rows behind the last among them."""
    rng = np.random.default_rng(heads + dim)
    for tokens, pairs in ((3, False), (257, True)):
        for in_place in (False, True) if heads else (False,):
            say("store size", dtype, heads, kv, dim, tokens, in_place)
            store(ctx, rng, dtype, tokens, heads, kv, dim, 64, 8, pairs ^ in_place, 1000, in_place, behind=2)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("pairs", [False, True])
def test_store_of_a_prompt(ctx, dtype, pairs):
    """300 tokens of 32 query and 8 key heads of 128, all of them rotated."""
    say("store prompt", dtype, pairs)
    store(ctx, np.random.default_rng(9), dtype, 300, 32, 8, 128, 16, 64, pairs, 5000, behind=1)


@pytest.mark.parametrize("heads,kv", [(12, 2), (28, 2), (32, 8), (64, 8), (113, 8)])
@pytest.mark.parametrize("dtype", [DT.F16, DT.Q8_0])
def test_store_errors_of_many_tokens(ctx, dtype, heads, kv):
    """Tokens with an error among sound ones, in every kernel: they keep their places, and the first is named."""
    dim, tokens = 128, 257
    rng = np.random.default_rng(heads)
    x = rng.standard_normal((tokens, heads + 2 * kv, dim)).astype(np.float32)
    bad = {40: (heads + 2 * kv - 1, 127), 41: (0, 0), 200: (heads, 50), 256: (heads + kv, 33)}
    for t, (h, e) in bad.items():
        x[t, h, e] = np.nan
    positions, freqs = cuda(np.arange(tokens, dtype=np.int32)), cuda(np.full(8, 0.01, np.float32))
    for n in (60, tokens):  # (as many tokens as CUs at most, and more)
        say("store errors", dtype, heads, kv, n)
        y = cuda(x[:n])
        cache, clean = (rlq.KvCache.make(dtype, 17, kv, 16, dim) for _ in range(2))
        out, want = (torch.full((n, heads, dim), 8.0, device="cuda") for _ in range(2))
        slots = np.arange(n) + 3
        args = y[:, heads:heads + kv], y[:, heads + kv:]
        ctx.kv_store(cache, *args, cuda(slots), y[:, :heads], positions[:n], freqs, out=out)
        h, e = bad[40]
        with raises("NonFiniteInput", h * dim + e, 40):
            ctx.sync()
        slots[[t for t in bad if t < n]] = -1
        ctx.kv_store(clean, *args, cuda(slots), y[:, :heads], positions[:n], freqs, out=want)
        ctx.sync()
        assert torch.equal(cache.k, clean.k) and torch.equal(cache.v, clean.v) and torch.equal(out, want)
        assert (out[40:42] == 8).all() and not (out[42] == 8).all()
