"""Attention over a paged cache: stored values at the ends of what the cache's types hold, many small weights, and rows beside
others."""
import numpy as np
import pytest

import kv_oracle as K
from rlq_loader import load
from test_gpu_kv import cuda, fill, say, tolerance

pytestmark = pytest.mark.gpu

rlq = load()
DT = rlq.DType
U = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module")
def ctx():
    c = rlq.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("scale", [511.5, 511.75, 512.0, 513.0, 515.5, 516.0, 65504.0])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
def test_attention_of_the_lowest_level(ctx, dim, scale):
    """A level is any int8: -128 times a scale of 512 is beyond f16, and a finite value of the cache all the same."""
    say("attention level -128", dim, scale)
    rng = np.random.default_rng(dim)
    rows, heads, kv, page, width = 3, 6, 2, 16, 10
    cache = rlq.KvCache.make(DT.Q8_0, rows * width, kv, page, dim)
    planes = []
    for t in (cache.k, cache.v):
        levels = rng.integers(-128, 128, (rows * width, kv, page * dim)).astype(np.int8)
        levels[rng.random(levels.shape) < 0.1] = -128
        scales = np.full((rows * width, kv, page * dim // 32), scale, np.float16)
        scales[rng.random(scales.shape) < 0.5] = 1.0
        b = np.concatenate([levels.view(np.uint8), scales.view(np.uint8)], -1)
        t.copy_(cuda(b))
        planes.append(K.values(b, True, page, dim))
    tables = rng.permutation(rows * width).astype(np.int32).reshape(rows, width)
    positions = np.array([width * page - 1, 40, 0], np.int32)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    factor = 0.01 / scale
    want, spread, most = K.attention(*planes, q, tables, positions, None, factor, 0, np.zeros_like(q))
    got = ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions), scale=factor)
    ctx.sync()
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tolerance(dim, spread, most) + U * np.abs(want)).all(), err.max()


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_attention_of_many_small_weights(ctx, dtype):
    """Every 32nd token takes nearly all of the weight and has no value, the others have value 1 and weights of 2^-32 to 2^-28
    of that: the result is the sum of those.

    Worst case of f32, relative to the result: a score (33 at most, to base 2) is off by nine roundings (its query times
    scale, the query's terms, four partial sums, the difference to the maximum), 9 * 33 * U * ln 2 = 1.2e-5; a weight by half of
    f16's least step, 2^-39 of the largest one's, up or down, so that 10000 of them are by five standard deviations
    4.1e-5 of the sum; the sum itself by some 100 roundings, 6e-6.  1e-4 is beyond all of them, and weights cut towards zero
    would be off by 1.4e-3."""
    say("attention small weights", dtype)
    rng = np.random.default_rng(77)
    n, heads, dim, page = 20001, 4, 64, 64
    width = -(-n // page)
    cache = rlq.KvCache.make(dtype, width, 1, page, dim)
    far = -rng.uniform(28, 32, width * page) * np.log(2)
    far[::32] = 0
    if dtype == DT.Q8_0:
        d = rng.uniform(0.2, 0.25, width * page).astype(np.float16)
        kl, vl = (np.zeros((width * page, dim), np.int8) for _ in range(2))
        kl[:, 0], kl[:, 1], vl[:] = np.round(far / d), rng.integers(-128, 128, width * page), 64
        kl[::32, 1], vl[::32] = 0, 0
        ks, vs = np.repeat(d[:, None], dim // 32, 1), np.full((width * page, dim // 32), 2.0 ** -6, np.float16)
        planes = []
        for t, levels, scales in ((cache.k, kl, ks), (cache.v, vl, vs)):
            b = np.concatenate([levels.reshape(width, 1, -1).view(np.uint8), scales.reshape(width, 1, -1).view(np.uint8)], -1)
            t.copy_(cuda(b))
            planes.append(K.values(b, True, page, dim))
    else:
        k, v = (np.zeros((width * page, dim), np.float32) for _ in range(2))
        k[:, 0], k[:, 1], v[:] = far, rng.uniform(-1, 1, width * page), 1
        k[::32, 1], v[::32] = 0, 0
        for t, x in ((cache.k, k), (cache.v, v)):
            t.copy_(cuda(x.reshape(width, 1, page, dim), t.dtype))
        planes = [t.double().cpu().numpy() for t in (cache.k, cache.v)]
    q = np.zeros((2, heads, dim), np.float32)
    q[..., 0], q[..., 1] = 1 - np.arange(heads) / 64, 2.0 ** -7
    tables, positions = np.arange(width, dtype=np.int32).reshape(1, -1), np.array([n - 1, n // 2], np.int32)
    requests = np.zeros(2, np.int32)
    want, _, _ = K.attention(*planes, q, tables, positions, requests, 1.0, 0, np.zeros_like(q))
    got = ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions), cuda(requests), 1.0)
    ctx.sync()
    err = np.abs(got.double().cpu().numpy() / want - 1)
    print("relative error", err.max(), flush=True)
    assert err.max() <= 1e-4


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_attention_of_rows_in_one_tile_does_not_depend_on_company(ctx, dtype):
    """Rows whose tokens lie within one aligned 128 of the positions, alone and beside long rows, runs of rows that go together
    and rows of other requests: the same bits."""
    say("attention company", dtype)
    rng = np.random.default_rng(31)
    heads, kv, dim, page, width = 8, 2, 64, 16, 640
    cache = rlq.KvCache.make(dtype, 2 * width, kv, page, dim)
    fill(rng, cache)
    tables = cuda(rng.permutation(2 * width).astype(np.int32).reshape(2, width))
    for window, positions in ((0, [0, 1, 30, 31, 32, 33, 100, 125, 126, 127]), (20, [19, 127, 147, 148, 149, 150, 151, 255, 9000, 9001])):
        first = [max(0, p + 1 - window) if window else 0 for p in positions]
        assert all(f >> 7 == p >> 7 for f, p in zip(first, positions))
        long = [5000, 10000, 128, 129, 130, 131, 132, 8000, 8001, 8002] * 20
        n = len(positions)
        q = cuda(rng.standard_normal((n + len(long), heads, dim)).astype(np.float32))
        at = cuda(np.array(positions + long, np.int32))
        who = cuda(np.concatenate([np.zeros(n), np.arange(len(long)) // 10 % 2]).astype(np.int32))
        for rows in (n, n + 10, n + len(long)):  # (few: counted by lanes; many: in LDS)
            together = ctx.kv_attention(cache, q[:rows], tables, at[:rows], who[:rows], window=window)
            for r in range(n):
                alone = ctx.kv_attention(cache, q[r:r + 1], tables, at[r:r + 1], who[r:r + 1], window=window)
                assert (alone[0] == together[r]).all(), (window, rows, r)
        ctx.sync()


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_attention_of_one_token_is_its_value(ctx, dtype, dim):
    """The weight of a token alone is 1 whatever its score, so its value comes out bit for bit: rows of one token, and rows that
    a window leaves one."""
    say("attention one token", dtype, dim)
    rng = np.random.default_rng(dim)
    rows, heads, kv, page, width = 200, 8, 2, 16, 12
    cache = rlq.KvCache.make(dtype, rows * width, kv, page, dim)
    _, v = fill(rng, cache)
    tables = rng.permutation(rows * width).astype(np.int32).reshape(rows, width)
    q = (rng.standard_normal((rows, heads, dim)) * rng.uniform(0.1, 8, (rows, 1, 1))).astype(np.float32)
    for window, positions in ((0, np.zeros(rows, np.int32)), (1, rng.integers(0, width * page, rows).astype(np.int32))):
        got = ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions), window=window)
        ctx.sync()
        want = v[tables[np.arange(rows), positions // page], :, positions % page].astype(np.float32)  # [rows, kv heads, dim]
        assert np.array_equal(got.cpu().numpy(), np.repeat(want, heads // kv, 1))
