"""Attention over a paged cache whose stored values lie at the ends of what the cache's types hold."""
import numpy as np
import pytest

import kv_oracle as K
from rlq_loader import load
from test_gpu_kv import cuda, say, tolerance

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
