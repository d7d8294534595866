"""rlq_kv_store: the place that an error names, within the four values of a thread too, and slots named twice."""
import numpy as np
import pytest

from rlq_loader import load
from test_gpu_kv import cuda, raises, say

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
