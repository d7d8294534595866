"""The paged KV cache on the GPU (rlq_kv_pages, rlq_kv_store, rlq_kv_attention) against
plain 64-bit forms: lengths from nothing to several splits, page borders, windows,
head layouts, strides, rows behind the last, errors among sound rows, other streams and
replayed graphs."""
import numpy as np
import pytest

import kv_oracle as K
from rlq_loader import load

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType
TORCH = {} if torch is None else {DT.F32: torch.float32, DT.F16: torch.float16, DT.BF16: torch.bfloat16}
U = 2.0 ** -24  # half a step of f32


def say(*a):
    print("[case]", *a, flush=True)


@pytest.fixture(scope="module")
def ctx():
    c = rlq.Context(0)
    yield c
    c.close()


def raises(name, a=None, b=None):
    class Check:
        def __enter__(self):
            return self

        def __exit__(self, kind, e, tb):
            assert kind is not None and issubclass(kind, rlq.QuantError), kind
            assert e.name == name and (a is None or e.a == a) and (b is None or e.b == b), e
            return True
    return Check()


def cuda(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).cuda()


def fill(rng, cache, size=1.0):
    """Random contents of a cache; returns them as f64 [pages, kv_heads, page, dim] pairs."""
    out = []
    for t in (cache.k, cache.v):
        shape = (cache.pages, cache.kv_heads, cache.page, cache.dim)
        x = (rng.standard_normal(shape) * size).astype(np.float32)
        if cache.dtype == DT.Q8_0:
            q, d = K.q8_0(x)
            b = np.concatenate([q.reshape(*shape[:2], -1).view(np.uint8), d.reshape(*shape[:2], -1).view(np.uint8)], -1)
            t.copy_(cuda(b))
            out.append(K.values(b, True, cache.page, cache.dim))
        else:
            t.copy_(cuda(x, TORCH[cache.dtype]))
            out.append(t.double().cpu().numpy())
    return out


def tolerance(dim, spread, most):
    """The f32 arithmetic's worst case: a score is a sum of dim products (at most dim + 2
    roundings of partial sums, each within U of sum|q k|, and the operands' splits within
    2^-22 of each product), an exponential is within 4 units, a sum over tokens and its
    joins at most doubles what its weights are off by (numerator and denominator) and adds
    64 roundings of |v|'s size."""
    score = (dim + 8) * U * spread + 8 * U
    return ((2 * score + 64 * U) * most)[..., None]


def attend(ctx, rng, dtype, rows, heads, kv, dim, page, longest, window=0, scale=None, positions=None, requests=None,
           table_rows=None, even=False, spread_pages=1, size=1.0):
    table_rows = table_rows or rows
    width = max(1, -(-max(longest, 1) // page))
    pool = table_rows * width
    if spread_pages > 1:  # pages that lie apart in a larger tensor
        base = [torch.zeros((pool, spread_pages, kv, page, dim), dtype=TORCH[dtype], device="cuda") for _ in range(2)]
        cache = rlq.KvCache(base[0][:, 1], base[1][:, 0], dtype, page, dim)
    else:
        cache = rlq.KvCache.make(dtype, pool, kv, page, dim)
    k, v = fill(rng, cache, size)
    tables = rng.permutation(pool).astype(np.int32).reshape(table_rows, width)
    if positions is None:
        positions = np.full(rows, longest - 1) if even else rng.integers(-1, longest, rows)
        positions[0] = longest - 1
    positions = np.asarray(positions, np.int32)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    out = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    req = None if requests is None else np.asarray(requests, np.int32)
    want, spread, most = K.attention(k, v, q, tables, positions, req, scale or dim ** -0.5, window, out)
    got = ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions), None if req is None else cuda(req), scale, window,
                           out=cuda(out))
    ctx.sync()
    got = got.double().cpu().numpy()
    err = np.abs(got - want)
    assert (err <= tolerance(dim, spread, most) + U * np.abs(want)).all(), (err.max(), np.unravel_index(err.argmax(), err.shape))
    live = spread.sum(1) > 0
    if live.any():  # independent roundings of a score are about U times its terms' sum, far below the worst case
        assert np.linalg.norm(err[live]) <= (3e-6 + 2 * U * spread.max()) * np.linalg.norm(want[live])
    return cache, q, tables, positions, got


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_types_and_dims(ctx, dtype, dim):
    say("attention", dtype, dim)
    rng = np.random.default_rng(dim + dtype)
    for heads, kv, page, longest in ((4, 2, 16, 77), (7, 1, 32, 300)):
        attend(ctx, rng, dtype, 5, heads, kv, dim, page, longest)


@pytest.mark.parametrize("longest", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000])
@pytest.mark.parametrize("dtype", [DT.F16, DT.Q8_0])
def test_attention_lengths(ctx, dtype, longest):
    say("attention length", dtype, longest)
    attend(ctx, np.random.default_rng(longest), dtype, 3, 8, 2, 64, 16, longest, even=True)


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 5), (32, 8), (14, 2), (16, 1), (17, 1), (33, 1), (71, 1), (40, 2), (48, 3)])
@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32])
def test_attention_head_layouts(ctx, dtype, heads, kv):
    say("attention heads", dtype, heads, kv)
    attend(ctx, np.random.default_rng(heads), dtype, 4, heads, kv, 64, 32, 150)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_attention_pages_and_windows(ctx, dtype, page):
    rng = np.random.default_rng(page)
    for window in (1, 2, 16, 33, 100, 700, 5000):
        say("attention window", dtype, page, window)
        attend(ctx, rng, dtype, 6, 8, 2, 64, page, 600, window=window)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_attention_long_rows_are_split(ctx, dtype):
    say("attention long", dtype)
    rng = np.random.default_rng(3)
    attend(ctx, rng, dtype, 1, 8, 2, 128, 64, 20000)
    attend(ctx, rng, dtype, 3, 4, 1, 64, 16, 9001, positions=[9000, 17, 4500])
    attend(ctx, rng, dtype, 2, 8, 8, 32, 128, 7000, window=6001)


@pytest.mark.parametrize("lengths", [(100, 256 * 128), (100, 256 * 128 - 127), (129, 384 * 128), (100, 255 * 128 + 1, 384 * 128, 300),
                                     (1, 128 * 128), (1, 17 * 128, 16 * 128)])
def test_attention_rows_that_begin_inside_a_slot(ctx, lengths):
    """A row of as many tiles as its parts may have, behind others: its first and last part are not whole."""
    say("attention inside", lengths)
    rng = np.random.default_rng(len(lengths))
    for kv in (1, 2):
        attend(ctx, rng, DT.F16, len(lengths), 2 * kv, kv, 32, 256, max(lengths), positions=np.asarray(lengths) - 1)


def test_attention_rows_of_few_and_many_requests(ctx):
    rng = np.random.default_rng(8)
    say("attention: tokens of a prompt")
    attend(ctx, rng, DT.F16, 100, 8, 2, 64, 16, 100, positions=np.arange(100), requests=np.zeros(100), table_rows=1)
    say("attention: five drafted tokens of each request, rows behind the last")
    positions = np.concatenate([np.arange(n - 5, n) for n in (5, 90, 33, 200)] + [[-1, 7, 300]])
    requests = np.concatenate([np.repeat([2, 0, 3, 1], 5), [-1, -1, -1]])
    attend(ctx, rng, DT.BF16, 23, 14, 2, 64, 32, 200, positions=positions, requests=requests, table_rows=4)
    say("attention: 700 requests, some without a token")
    attend(ctx, rng, DT.F16, 700, 4, 1, 32, 16, 40)
    say("attention: nobody has a token")
    _, _, _, _, got = attend(ctx, rng, DT.F16, 3, 4, 2, 32, 16, 40, positions=[-1, -1, -1])
    assert (got == 0).all()


@pytest.mark.parametrize("rows", [63, 64, 65, 255, 1023, 1024, 1025, 2100])
def test_attention_row_counts(ctx, rows):
    """Rows counted by lanes, in LDS, and over several launches; with and without requests, empty rows among them."""
    say("attention rows", rows)
    rng = np.random.default_rng(rows)
    attend(ctx, rng, DT.F16, rows, 2, 1, 32, 16, 20)
    positions = np.where(np.arange(rows) % 7 == 0, -1, rng.integers(0, 300, rows))
    requests = np.where(np.arange(rows) % 11 == 0, -1, np.arange(rows) % 3)
    attend(ctx, rng, DT.F16, rows, 2, 1, 32, 16, 300, positions=positions, requests=requests, table_rows=3)


def test_attention_at_the_last_position(ctx):
    """A position at the end of 32 bits: a window over the last pages of a table that names few."""
    say("attention last position")
    cache = rlq.KvCache.make(DT.F16, 3, 1, 256, 32)
    k, v = fill(np.random.default_rng(1), cache)
    width = 2 ** 31 // 256
    tables = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    tables[0, -2:] = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    q = np.random.default_rng(2).standard_normal((1, 2, 32)).astype(np.float32)
    last = 2 ** 31 - 1
    got = ctx.kv_attention(cache, cuda(q), tables, cuda(np.array([last], np.int32)), window=300)
    ctx.sync()
    flat = [x[[2, 1], 0].reshape(512, 32)[-300:] for x in (k, v)]
    s = flat[0] @ q[0].T.astype(np.float64) * 32 ** -0.5
    p = np.exp(s - s.max(0))
    want = (p / p.sum(0)).T @ flat[1]
    assert np.abs(got[0].cpu().numpy() - want).max() <= 1e-5  # (32 products and 300 weights in f32: 2^-24 (40 + 64) |v|)
    ctx.kv_attention(cache, cuda(q), tables, cuda(np.array([last], np.int32)), window=600)
    with raises("Bounds", 0):
        ctx.sync()


def test_attention_far_scores_and_scales(ctx):
    """Scores that spread over hundreds (one token has all the weight), a scale of its own, negative too."""
    rng = np.random.default_rng(4)
    for dtype in (DT.F32, DT.F16, DT.BF16, DT.Q8_0):
        for scale in (3.0, 0.001, -0.5):
            say("attention scale", dtype, scale)
            attend(ctx, rng, dtype, 3, 4, 2, 64, 16, 200, scale=scale)


@pytest.mark.parametrize("dtype,size", [(DT.F16, 1e-6), (DT.F16, 1e4), (DT.BF16, 1e-30), (DT.BF16, 1e20), (DT.F32, 1e-30),
                                        (DT.F32, 1e15), (DT.Q8_0, 1e-3), (DT.Q8_0, 1e4), (DT.Q8_0, 1e6)])
def test_attention_of_small_and_large_values(ctx, dtype, size):
    """Keys and values of f16's subnormal range, near the types' ends, and 8-bit blocks whose scales are
    f16 subnormals, beyond 515 (where level times scale leaves f16), or near f16's largest."""
    say("attention value size", dtype, size)
    rng = np.random.default_rng(14)
    for dim in (64, 96):
        attend(ctx, rng, dtype, 3, 6, 2, dim, 16, 150, scale=0.1 / size, size=size)


def test_attention_of_scales_beyond_f16(ctx):
    """Blocks with a value beyond 127 times f16's largest have an infinite scale: no finite result, and said so."""
    say("attention infinite scales")
    with raises("NonFinite", 6), np.errstate(all="ignore"):
        attend(ctx, np.random.default_rng(14), DT.Q8_0, 3, 6, 2, 64, 16, 150, scale=0.1 / 2e6, size=2e6)


@pytest.mark.parametrize("dtype", [DT.F16, DT.BF16, DT.F32])
@pytest.mark.parametrize("size", [1e-5, 1e4])
def test_attention_small_and_large_queries(ctx, dtype, size):
    """Queries far from 1, with keys that bring the scores back."""
    say("attention query size", dtype, size)
    rng = np.random.default_rng(5)
    cache = rlq.KvCache.make(dtype, 4, 1, 16, 64)
    k, v = fill(rng, cache)
    q = (rng.standard_normal((2, 4, 64)) * size).astype(np.float32)
    tables, positions = np.arange(4, dtype=np.int32).reshape(1, 4), np.array([50, 63], np.int32)
    requests = np.zeros(2, np.int32)
    want, spread, most = K.attention(k, v, q, tables, positions, requests, 0.125 / size, 0, np.zeros_like(q))
    got = ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions), cuda(requests), 0.125 / size)
    ctx.sync()
    assert (np.abs(got.cpu().numpy() - want) <= tolerance(64, spread, most)).all()


def test_attention_strides_and_pages_that_lie_apart(ctx):
    rng = np.random.default_rng(6)
    say("attention strides")
    for dtype in (DT.F16, DT.F32):
        attend(ctx, rng, dtype, 4, 6, 3, 64, 16, 100, spread_pages=3)
    cache, q, tables, positions, got = attend(ctx, rng, DT.F16, 4, 6, 3, 64, 16, 100)
    fused = torch.zeros((4, 12, 64), device="cuda")
    fused[:, :6] = cuda(q)
    wide = torch.full((4, 9, 64), 7.0, device="cuda")
    ctx.kv_attention(cache, fused[:, :6], cuda(tables), cuda(positions), out=wide[:, 2:8])
    ctx.sync()
    assert np.array_equal(wide[:, 2:8].cpu().numpy(), got)
    assert (wide[:, :2] == 7).all() and (wide[:, 8] == 7).all()
    # rows that are 4-byte aligned only
    odd = torch.zeros(4 * 6 * 64 + 1, device="cuda")[1:].view(4, 6, 64)
    odd.copy_(cuda(q))
    assert np.array_equal(ctx.kv_attention(cache, odd, cuda(tables), cuda(positions)).cpu().numpy(), got)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16])
def test_attention_does_not_look_at_masked_places(ctx, dtype):
    """NaN and infinities behind the last token, before the window, in other pages and heads."""
    say("attention masked", dtype)
    rng = np.random.default_rng(7)
    cache = rlq.KvCache.make(dtype, 40, 2, 16, 64)
    k, v = fill(rng, cache)
    q = cuda(rng.standard_normal((3, 4, 64)).astype(np.float32))
    tables = cuda(rng.permutation(39).astype(np.int32)[:36].reshape(3, 12))
    positions = [100, 37, 64]
    for window in (0, 30):
        pos = cuda(np.array(positions, np.int32))
        want = ctx.kv_attention(cache, q, tables, pos, window=window).clone()
        ctx.sync()
        dirty = rlq.KvCache(cache.k.clone(), cache.v.clone(), dtype, 16, 64)
        for t, bad in ((dirty.k, float("nan")), (dirty.v, float("inf"))):
            keep = torch.zeros((40, 16), dtype=torch.bool, device="cuda")
            for r, p in enumerate(positions):
                at = torch.arange(max(0, p + 1 - window) if window else 0, p + 1, device="cuda")
                keep[tables[r, at // 16].long(), at % 16] = True
            t.copy_(torch.where(keep[:, None, :, None], t, torch.full_like(t, bad)))
        got = ctx.kv_attention(dirty, q, tables, pos, window=window)
        ctx.sync()
        assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 2), (3, 1), (8, 2), (5, 1), (14, 2), (16, 2), (9, 1), (34, 2)])
@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
def test_attention_of_runs_of_rows(ctx, dtype, heads, kv):
    """Rows of a request at one position after the other, in runs of all lengths, that end and begin anywhere; with rows
    without a token, gaps, steps back and other requests between them."""
    say("attention runs", dtype, heads, kv)
    rng = np.random.default_rng(heads)
    positions, requests = [], []
    for n in (1, 2, 3, 4, 5, 7, 16, 17, 3):
        start, r = int(rng.integers(0, 270)), int(rng.integers(0, 3))
        positions += range(start, start + n)
        requests += [r] * n
    positions += [-1, 0, 1, 2, 2, 1, 4, 126, 127, 128, 129, 299]
    requests += [1, 1, 1, 1, 1, 1, 1, 2, 2, 2, 2, -1]
    for window in (0, 1, 40):  # (many heads or rows: they go together where there is more to do than the CUs hold)
        attend(ctx, rng, dtype, len(positions), 8 * heads, 8 * kv, 64, 16, 300, window=window, positions=positions,
               requests=requests, table_rows=3)
        n = 7 * len(positions)
        attend(ctx, rng, dtype, n, heads, kv, 32, 32, 300, window=window, positions=positions * 7, requests=requests * 7,
               table_rows=3)


@pytest.mark.parametrize("dtype", [DT.F16, DT.BF16, DT.Q8_0])
def test_attention_of_long_runs(ctx, dtype):
    """Runs over several slots; rows of a prompt that is longer than a launch's rows."""
    say("attention long runs", dtype)
    rng = np.random.default_rng(20)
    positions = np.concatenate([n - 5 + np.arange(5) for n in (20000, 9000, 130, 257)])
    attend(ctx, rng, dtype, 20, 8, 2, 128, 64, 20000, positions=positions, requests=np.repeat(np.arange(4), 5), table_rows=4)
    attend(ctx, rng, dtype, 1500, 2, 1, 32, 16, 1600, positions=100 + np.arange(1500), requests=np.zeros(1500), table_rows=1)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("start", [20, 125])
def test_attention_of_runs_keeps_rows_apart(ctx, dtype, start):
    """A value or key that is no number, or a page that is none, is the error of the rows that see it."""
    rng = np.random.default_rng(start)
    dim, page, n, heads = 64, 16, 6, 256  # (so many that rows go together); KV head 1 is that of heads 2 and 3
    for window in (0, 10):
        cache, q, tables, positions, got = attend(ctx, rng, dtype, n, heads, heads // 2, dim, page, 160, window=window,
                                                  positions=start + np.arange(n), requests=np.zeros(n), table_rows=1)
        req = cuda(np.zeros(n, np.int32))

        def call(t, held, name, a, free=lambda r, h: False):
            out = torch.full((n, heads, dim), 5.0, device="cuda")
            ctx.kv_attention(cache, cuda(q), cuda(t), cuda(positions), req, window=window, out=out)
            with raises(name, *a):
                ctx.sync()
            out = out.cpu().numpy()
            for r in range(n):
                for h in range(heads):
                    if free(r, h):
                        assert np.isfinite(out[r, h]).all() and (out[r, h] != 5).all()
                        continue
                    assert (out[r, h] == 5).all() if held(r, h) else np.array_equal(out[r, h], got[r, h]), (r, h)

        for plane in (cache.k, cache.v):
            for token, rows in ((start + 3, range(3, n)), (start - 9, [0] if window else range(n)), (start + n - 1, [n - 1])):
                say("attention runs apart", dtype, window, token)
                where = plane[int(tables[0, token // page]), 1]
                kept = where.clone()
                low = np.zeros((n, heads), bool)
                if dtype == DT.Q8_0:  # an infinite scale
                    where[page * dim:].view(torch.float16)[(token % page) * (dim // 32)] = float("inf")
                    if plane is cache.k:  # a score of -infinity where the block's product is negative: a weight of 0
                        levels = where[token % page * dim:][:32].view(torch.int8).double().cpu().numpy()
                        low = q[..., :32] @ levels < 0
                else:
                    where[token % page, 5] = float("nan")
                sees = [(r, h) for r in rows for h in (2, 3)]
                off = [r for r, h in sees if not low[r, h]]
                if off:
                    call(tables, lambda r, h: (r, h) in sees, "NonFinite", (6, off[0]), lambda r, h: (r, h) in sees and low[r, h])
                where.copy_(kept)
        if start % page + n > page:  # the last rows' page is none
            t = tables.copy()
            t[0, start // page + 1] = -1
            first = page * (start // page + 1) - start
            call(t, lambda r, h: r >= first, "Bounds", (first,))


def test_attention_errors_are_the_rows_own(ctx):
    say("attention errors")
    rng = np.random.default_rng(9)
    cache, q, tables, positions, got = attend(ctx, rng, DT.F16, 6, 4, 2, 64, 16, 90, positions=[89, 40, 20, 89, 0, 88])
    for change, name, row in ((lambda t, p, x: t.__setitem__((1, 2), 36), "Bounds", 1),
                              (lambda t, p, x: t.__setitem__((3, 5), -1), "Bounds", 3),
                              (lambda t, p, x: p.__setitem__(4, 96), "Bounds", 4),
                              (lambda t, p, x: p.__setitem__(2, -2), "Bounds", 2),
                              (lambda t, p, x: x.__setitem__((5, 1, 3), np.nan), "NonFinite", 5),
                              (lambda t, p, x: x.__setitem__((0, 3, 0), np.inf), "NonFinite", 0)):
        t, p, x = tables.copy(), positions.copy(), q.copy()
        change(t, p, x)
        out = torch.full((6, 4, 64), 5.0, device="cuda")
        ctx.kv_attention(cache, cuda(x), cuda(t), cuda(p), out=out)
        with raises(name, *((row,) if name == "Bounds" else (6, row))):
            ctx.sync()
        ctx.sync()  # (reported once)
        others = [r for r in range(6) if r != row]
        assert np.array_equal(out[others].cpu().numpy(), got[others])
        held = range(4) if name == "Bounds" else [1] if row == 5 else [3]
        for h in range(4):  # (heads of the row that are not concerned are written)
            assert (out[row, h] == 5).all() if h in held else np.array_equal(out[row, h].cpu().numpy(), got[row, h])
    # a column that no row needs may hold anything
    t = tables.copy()
    t[2, 3], t[1, 5] = -7, 10 ** 6
    out = ctx.kv_attention(cache, cuda(q), cuda(t), cuda(positions))
    ctx.sync()
    assert np.array_equal(out.cpu().numpy(), got)
    requests = np.array([0, 1, 2, 6, -2, 5], np.int32)
    out = torch.full((6, 4, 64), 5.0, device="cuda")
    ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions), cuda(requests), out=out)
    with raises("Bounds", 3):
        ctx.sync()
    assert (out[3:5] == 5).all() and np.array_equal(out[[0, 1, 2, 5]].cpu().numpy(), got[[0, 1, 2, 5]])


def test_attention_is_the_same_every_time(ctx):
    """Splits are joined in one order: the same bits in every run."""
    say("attention repeated")
    rng = np.random.default_rng(10)
    cache, q, tables, positions, got = attend(ctx, rng, DT.F16, 5, 8, 2, 64, 16, 3000)
    for _ in range(10):
        assert np.array_equal(ctx.kv_attention(cache, cuda(q), cuda(tables), cuda(positions)).cpu().numpy(), got)
    ctx.sync()


# ---- store ----------------------------------------------------------------------------


def store(ctx, rng, dtype, tokens, heads, kv, dim, page, half, pairs, start=0, in_place=False, behind=0):
    pages = -(-tokens // page) + 3
    cache = rlq.KvCache.make(dtype, pages, kv, page, dim)
    fill(rng, cache)
    before = [t.clone() for t in (cache.k, cache.v)]
    fused = cuda(rng.standard_normal((tokens + behind, (heads + 2 * kv) * dim)).astype(np.float32))
    parts = [fused[:, :heads * dim].unflatten(1, (heads, dim)) if heads else None,
             fused[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim)),
             fused[:, (heads + kv) * dim:].unflatten(1, (kv, dim))]
    q, k, v = (None if t is None else t.cpu().numpy().copy() for t in parts)
    positions = (np.arange(tokens + behind) + start).astype(np.int32)
    slots = np.concatenate([rng.permutation(pages * page)[:tokens], np.full(behind, -1)]).astype(np.int64)
    freqs = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
    out = parts[0] if in_place else None if q is None else torch.full((tokens + behind, heads, dim), 3.0, device="cuda")
    got = ctx.kv_store(cache, parts[1], parts[2], cuda(slots), parts[0], cuda(positions), cuda(freqs) if half else None, pairs, out)
    ctx.sync()
    n = tokens
    if heads:
        want = K.rotate(q, positions, freqs, pairs)
        want[n:] = q[n:] if in_place else 3.0
        # (the last bit of an f64 sine may turn a rounding to f32: one such value in 2^28 or so)
        assert np.array_equal(got.cpu().numpy(), want)
    for t, old, x in zip((cache.k, cache.v), before, (K.rotate(k, positions, freqs, pairs), v)):
        want = old.cpu()
        p, o = slots[:n] // page, slots[:n] % page
        if dtype == DT.Q8_0:
            levels, scales = K.q8_0(x[:n])
            want = want.numpy()
            lv = want[..., :page * dim].view(np.int8).reshape(pages, kv, page, dim)
            sc = np.ascontiguousarray(want[..., page * dim:]).view(np.float16).reshape(pages, kv, page, dim // 32)
            lv = lv.copy()
            lv[p, :, o], sc[p, :, o] = levels, scales
            want = torch.from_numpy(np.concatenate([lv.reshape(pages, kv, -1).view(np.uint8),
                                                    sc.reshape(pages, kv, -1).view(np.uint8)], -1))
        else:
            want[p, :, o] = torch.from_numpy(x[:n]).to(TORCH[dtype])
        assert torch.equal(t.cpu(), want)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("heads,kv,dim,half,pairs", [
    (32, 8, 128, 64, True), (14, 2, 64, 32, False), (4, 4, 32, 16, True), (6, 3, 96, 24, False), (5, 1, 96, 48, True),
    (3, 1, 160, 80, False), (2, 2, 192, 96, True), (2, 1, 224, 112, False), (8, 2, 256, 128, False), (4, 2, 256, 128, True),
    (4, 2, 64, 1, True), (4, 2, 64, 7, False), (4, 2, 128, 0, True), (0, 2, 64, 32, True), (100, 2, 64, 32, False)])
def test_store(ctx, dtype, heads, kv, dim, half, pairs):
    rng = np.random.default_rng(dim + half)
    for tokens, page, start, behind in ((1, 16, 0, 0), (5, 32, 1000, 2), (67, 64, 1000000, 1)):
        say("store", dtype, heads, kv, dim, half, pairs, tokens)
        store(ctx, rng, dtype, tokens, heads, kv, dim, page, half, pairs, start, behind=behind)
        if heads:
            store(ctx, rng, dtype, tokens, heads, kv, dim, page, half, pairs, start, in_place=True, behind=behind)


@pytest.mark.parametrize("tokens", [1, 3, 64, 1000])
def test_store_many_tokens(ctx, tokens):
    say("store tokens", tokens)
    rng = np.random.default_rng(tokens)
    store(ctx, rng, DT.BF16, tokens, 8, 2, 64, 256, 32, False, 5)
    store(ctx, rng, DT.Q8_0, tokens, 8, 2, 64, 128, 32, True, 2 ** 31 - 1 - tokens)


def test_store_of_large_angles(ctx):
    """Angles beyond the polynomial's reduction, and just before it."""
    say("store large angles")
    rng = np.random.default_rng(3)
    cache = rlq.KvCache.make(DT.F32, 1, 1, 16, 64)
    k, v = (rng.standard_normal((8, 1, 64)).astype(np.float32) for _ in range(2))
    positions = np.array([2 ** 31 - 1, 2 ** 31 - 8, 10 ** 9 + 7, 3, 0, -5, -2 ** 31, 123456789], np.int32)
    freqs = np.geomspace(1e-7, 1e6, 32).astype(np.float32)
    ctx.kv_store(cache, cuda(k), cuda(v), cuda(np.arange(8)), positions=cuda(positions), freqs=cuda(freqs), pairs=False)
    ctx.sync()
    assert np.array_equal(cache.k[0, 0, :8].cpu().numpy(), K.rotate(k, positions, freqs, False)[:, 0])


def test_store_rounds_once(ctx):
    """Halfway values, subnormals and the largest value of each type; zero blocks of Q8_0."""
    say("store rounding")
    for dtype in (DT.F16, DT.BF16, DT.F32):
        t = TORCH[dtype]
        f = torch.finfo(t)
        steps = torch.tensor([1.0, 1 + f.eps / 2, 1 + f.eps, 1 + 1.5 * f.eps, f.max, -f.max, f.tiny, f.tiny * f.eps, 0.0, -0.0,
                              f.tiny * f.eps * 1.5 if dtype != DT.F32 else 1.0, 3.14159], dtype=torch.float64).float()
        x = steps.repeat(3)[:32].view(1, 1, 32).contiguous()
        cache = rlq.KvCache.make(dtype, 1, 1, 16, 32)
        ctx.kv_store(cache, x.cuda(), -x.cuda(), cuda(np.array([3])))
        ctx.sync()
        assert torch.equal(cache.k[0, 0, 3].cpu(), x[0, 0].to(t)) and torch.equal(cache.v[0, 0, 3].cpu(), -x[0, 0].to(t))
    cache = rlq.KvCache.make(DT.Q8_0, 1, 1, 16, 64)
    x = torch.zeros((1, 1, 64))
    x[0, 0, 40] = -254.0
    cache.k.fill_(9)
    ctx.kv_store(cache, x.cuda(), x.cuda(), cuda(np.array([15])))
    ctx.sync()
    b = cache.k[0, 0].cpu().numpy()
    levels, scales = b[:1024].view(np.int8).reshape(16, 64), b[1024:].view(np.float16).reshape(16, 2)
    assert levels[15, 40] == -127 and np.count_nonzero(levels[15]) == 1 and scales[15].tolist() == [0.0, 2.0]
    assert (b[:960] == 9).all()


def test_store_errors_are_the_tokens_own(ctx):
    say("store errors")
    rng = np.random.default_rng(2)
    x = [rng.standard_normal((4, n, 64)).astype(np.float32) for n in (4, 2, 2)]
    positions, freqs = cuda(np.arange(4, dtype=np.int32)), cuda(np.full(32, 0.01, np.float32))
    for dtype, part, value, name, a in (
            (DT.F16, 0, np.nan, "NonFiniteInput", None), (DT.F16, 1, np.inf, "NonFiniteInput", None),
            (DT.F16, 2, 70000.0, "NonFiniteInput", 4 * 64 + 2 * 64 + 64 + 40), (DT.BF16, 2, 3.4e38, "NonFiniteInput", 448 + 40),
            (DT.F32, 2, np.nan, "NonFiniteInput", 448 + 40), (DT.Q8_0, 2, np.nan, "NonFiniteInput", 448 + 40),
            (DT.Q8_0, 2, 1e8, "UnrepresentableScale", 7), (DT.F16, None, 48, "Bounds", 2), (DT.F16, None, -2, "Bounds", 2)):
        y = [t.copy() for t in x]
        slots = np.array([5, 17, 40, 3])
        if part is None:
            slots[2] = value
        else:
            y[part][2, 1, 40] = value
        cache = rlq.KvCache.make(dtype, 3, 2, 16, 64)
        clean = rlq.KvCache.make(dtype, 3, 2, 16, 64)
        out, want = (torch.full((4, 4, 64), 8.0, device="cuda") for _ in range(2))
        q, k, v = map(cuda, y)
        ctx.kv_store(cache, k, v, cuda(slots), q, positions, freqs, out=out)
        with raises(name, a, None if name == "Bounds" else 2):
            ctx.sync()
        slots[2] = -1
        ctx.kv_store(clean, k, v, cuda(slots), q, positions, freqs, out=want)
        ctx.sync()
        assert torch.equal(cache.k, clean.k) and torch.equal(cache.v, clean.v) and torch.equal(out, want)
        assert (out[2] == 8).all() and not (out[3] == 8).all()


# ---- pages ------------------------------------------------------------------------------


class Pages:
    """A cache's bookkeeping on both sides."""

    def __init__(self, requests, width, pages, page, seed, owned=False):
        rng = np.random.default_rng(seed)
        self.page, self.pages = page, pages
        self.tables = np.full((requests, width), -1, np.int32)
        self.owned = self.tables.copy() if owned else None
        self.free = rng.permutation(pages).astype(np.int32)
        self.count = np.array([pages], np.int32)
        self.lengths = np.zeros(requests, np.int32)
        self.on = {n: cuda(getattr(self, n)) for n in ("tables", "free", "count", "lengths")}
        self.on["owned"] = cuda(self.owned) if owned else None

    def step(self, ctx, new, tokens, in_place=True, stream=None):
        new = np.asarray(new, np.int32)
        o, n = self.on, len(self.lengths)
        i32 = dict(dtype=torch.int32, device="cuda")
        out = (o["lengths"], o["count"], torch.full((n + 1,), 9, **i32), torch.full((tokens,), 9, dtype=torch.int64, device="cuda"),
               torch.full((tokens,), 9, **i32), torch.full((tokens,), 9, **i32)) if in_place else None
        got = ctx.kv_pages(o["lengths"], cuda(new), o["tables"], o["free"], o["count"], self.page, tokens, o["owned"], out)
        ctx.sync()
        want = K.pages(self.lengths, new, self.tables, self.owned, self.free, self.count, self.page, tokens)
        for a, b in zip(got, want):
            assert np.array_equal(a.cpu().numpy(), b)
        for name in ("tables", "free", "owned"):
            if o[name] is not None:
                assert np.array_equal(o[name].cpu().numpy(), getattr(self, name)), name
        self.lengths, self.count = want[:2]
        o["lengths"], o["count"] = got[:2]
        return got


@pytest.mark.parametrize("requests,page,most", [(1, 16, 3), (3, 16, 40), (32, 32, 1), (200, 64, 300), (1000, 16, 5),
                                                (1025, 256, 20), (4096, 128, 3)])
@pytest.mark.parametrize("owned", [False, True])
def test_pages_over_steps(ctx, requests, page, most, owned):
    """Requests come, grow, wait and end; pages come back and are given out again."""
    rng = np.random.default_rng(requests)
    width = -(-most * 8 // page)
    p = Pages(requests, width, requests * width, page, 1, owned)
    for k in range(8):
        say("pages", requests, page, most, owned, "step", k)
        new = rng.integers(0, most + 1, requests)
        if k:
            new[rng.random(requests) < 0.2] = -1
        p.step(ctx, new, int(np.maximum(new, 0).sum()) + (5 if k % 2 else 0), in_place=k != 3)
    p.step(ctx, np.full(requests, -1), 0)
    assert p.count[0] == p.pages and sorted(p.free) == list(range(p.pages))


def test_pages_of_large_batches(ctx):
    say("pages: 60000 rows")
    p = Pages(50, 200, 10000, 16, 2)
    p.step(ctx, np.full(50, 1200), 60000)
    p.step(ctx, np.arange(50), 4097)
    p.step(ctx, np.r_[np.full(25, -1), np.full(25, 17)], 4096)


def test_pages_with_holes(ctx):
    """Entries of an ended request that are no page of its own (negative) stay off the list."""
    say("pages: holes")
    p = Pages(3, 8, 24, 16, 3, owned=True)
    p.step(ctx, [100, 20, 0], 120)
    p.owned[0, 2:4] = -1
    p.on["owned"].copy_(cuda(p.owned))
    p.step(ctx, [-1, 3, 5], 8)
    assert p.count[0] == 24 - 9 + 5 - 1


def test_pages_of_tokens_without_a_page(ctx):
    """A table whose part-filled page is missing: the slots say so, and the store reports them."""
    say("pages: a missing page")
    for tokens in (4, 5000):
        p = Pages(2, 4, 8, 16, 3)
        p.step(ctx, [20, 30], 50)
        p.on["tables"][0, 1] = -1
        _, _, _, slots, _, requests = ctx.kv_pages(p.on["lengths"], cuda(np.array([2, 1], np.int32)), p.on["tables"], p.on["free"],
                                                   p.on["count"], 16, tokens)
        ctx.sync()
        assert slots[:2].tolist() == [-2, -2] and slots[2] >= 0 and (slots[3:] == -1).all() and (requests[:3] >= 0).all()
        cache = rlq.KvCache.make(DT.F16, 8, 1, 16, 32)
        x = torch.ones((3, 1, 32), device="cuda")
        ctx.kv_store(cache, x, x, slots[:3].contiguous())
        with raises("Bounds", 0):
            ctx.sync()
        assert cache.k.sum() == 32


def test_pages_refusals(ctx):
    say("pages refusals")

    def refused(new, tokens, name, a, b=None, **set_):
        p = Pages(4, 4, 12, 16, 4)
        p.step(ctx, [30, 64, 0, 17], 120)
        for key, value in set_.items():
            p.on[key].copy_(cuda(np.asarray(value, np.int32)))
        state = {n: t.clone() for n, t in p.on.items() if t is not None}
        i32 = dict(dtype=torch.int32, device="cuda")
        out = [torch.full((n,), 9, **i32) for n in (4, 1, 5)] + [torch.full((tokens,), 9, dtype=torch.int64, device="cuda")] + \
              [torch.full((tokens,), 9, **i32) for _ in range(2)]
        ctx.kv_pages(p.on["lengths"], cuda(np.asarray(new, np.int32)), p.on["tables"], p.on["free"], p.on["count"], 16, tokens, None,
                     out)
        with raises(name, a, b):
            ctx.sync()
        for n, t in state.items():
            assert torch.equal(p.on[n], t), n
        assert all((t == 9).all() for t in out)

    for tokens in (64, 5000):  # (one launch, two launches)
        refused([1, 0, 60, 20], tokens, "InvalidState", 3, 1)       # 4 pages are left: no page for request 3's last
        refused([0, 1, 0, 0], tokens, "InvalidState", 1, 2)         # a fifth column
        refused([0, 0, 0, 0], tokens, "InvalidState", 2, 4, lengths=[30, 64, -1, 17])
        refused([0, 0, 2 ** 31 - 1, 0], tokens, "InvalidState", 2, 4, lengths=[30, 64, 1, 17])
        refused([0, 0, 0, 0], tokens, "InvalidState", 0, 0, count=[-1])
        refused([0, 0, 0, 0], tokens, "InvalidState", 0, 0, count=[13])
        refused([0, -1, 0, 0], tokens, "InvalidState", 0, 0, count=[9])  # 9 + 4 pages on a list of 12
        table = [[0, 1, 2, 3], [4, 5, 12, 7], [8, 9, 10, 11], [0, 1, 2, 3]]
        refused([0, -1, 0, 0], tokens, "Bounds", 6, tables=table)
    refused([1, 0, 2, 0], 2, "InvalidState", 2, 3)                  # three rows in a batch of two
    refused([1, 0, 0, 0], 0, "InvalidState", 0, 3)


# ---- together, streams, graphs ----------------------------------------------------------


def test_calls_in_a_captured_step(ctx):
    """A step's three calls recorded in a graph and replayed, with the lengths carried on
    the GPU, between eager calls: every replay against the same steps run eagerly."""
    say("captured step")
    rng = np.random.default_rng(11)
    n, heads, kv, dim, page, width = 6, 8, 2, 64, 16, 20

    def state():
        i32 = dict(dtype=torch.int32, device="cuda")
        s = {"tables": torch.full((n, width), -1, **i32), "free": torch.arange(n * width, **i32),
             "count": torch.full((1,), n * width, **i32), "lengths": torch.zeros(n, **i32),
             "cache": rlq.KvCache.make(DT.F16, n * width, kv, page, dim), "out": torch.zeros((n, heads, dim), device="cuda")}
        s["rows"] = (s["lengths"], s["count"], torch.zeros(n + 1, **i32), torch.zeros(n, dtype=torch.int64, device="cuda"),
                     torch.zeros(n, **i32), torch.zeros(n, **i32))
        s["x"] = torch.zeros((n, heads + 2 * kv, dim), device="cuda")
        s["q"] = torch.zeros((n, heads, dim), device="cuda")
        return s

    new = torch.ones(n, dtype=torch.int32, device="cuda")
    freqs = cuda((10000.0 ** (-np.arange(32) / 32)).astype(np.float32))

    def step(s):
        _, _, _, slots, positions, requests = ctx.kv_pages(s["lengths"], new, s["tables"], s["free"], s["count"], page, n, out=s["rows"])
        x = s["x"]
        ctx.kv_store(s["cache"], x[:, heads:heads + kv], x[:, heads + kv:], slots, x[:, :heads], positions, freqs, out=s["q"])
        ctx.kv_attention(s["cache"], s["q"], s["tables"], positions, requests, out=s["out"])

    a, b = state(), state()
    xs = [cuda(rng.standard_normal(tuple(a["x"].shape)).astype(np.float32)) for _ in range(60)]
    prompt = xs[0]
    for s in (a, b):
        s["x"].copy_(prompt)
        step(s)  # (the scratch is there)
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for i, x in enumerate(xs[1:]):
        a["x"].copy_(x)
        b["x"].copy_(x)
        graph.replay()
        step(b)
        if i % 7 == 0:
            torch.cuda.synchronize()
        for name in ("tables", "free", "count", "lengths", "out"):
            assert torch.equal(a[name], b[name]), (i, name)
        assert torch.equal(a["cache"].k, b["cache"].k) and torch.equal(a["cache"].v, b["cache"].v)
    ctx.sync()


def test_a_call_after_growth_leaves_recorded_ones_right(ctx):
    say("replay after growth")
    rng = np.random.default_rng(12)
    own = rlq.Context(0)
    cache, q, tables, positions, got = attend(own, rng, DT.F16, 2, 8, 2, 64, 16, 3000)
    args = cuda(q), cuda(tables), cuda(positions)
    out = torch.zeros((2, 8, 64), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        own.kv_attention(cache, *args, out=out)
    attend(own, rng, DT.F16, 600, 16, 4, 128, 16, 500)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), got)
    own.close()


def test_given_stream(ctx):
    say("given stream")
    rng = np.random.default_rng(13)
    cache, q, tables, positions, got = attend(ctx, rng, DT.F16, 3, 8, 2, 64, 16, 700)
    args = cuda(q), cuda(tables), cuda(positions)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for at in (s, s.cuda_stream, 0):
        out = ctx.kv_attention(cache, *args, stream=at)
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), got)
    ctx.sync()


@pytest.mark.parametrize("handle", [False, True], ids=["stream", "handle"])
@pytest.mark.parametrize("name", ["kv_pages", "kv_store", "kv_attention", "beam_select", "beam_reorder"])
def test_calls_on_a_given_stream_beside_a_busy_one(name, handle):
    """What a call makes is the given stream's, and it does not wait for torch's current one."""
    say("given stream, busy", name, handle)
    rng = np.random.default_rng(15)
    own = rlq.Context(0)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = rlq.KvCache.make(DT.F16, 40, 2, 16, 64)
    fill(rng, cache)
    x = cuda(rng.standard_normal((4, 8, 64)).astype(np.float32))
    slots, positions = cuda(np.array([3, 40, 77, 200])), cuda(np.array([90, 33, 5, 64], np.int32))
    tables, freqs = cuda(rng.permutation(40).astype(np.int32).reshape(4, 10)), cuda(np.full(32, 0.1, np.float32))
    logits, scores = cuda(rng.standard_normal((2, 2, 9000)).astype(np.float32)), torch.zeros((2, 2), device="cuda")
    lengths, new, free = cuda(np.array([5, 20, 0, 7], np.int32)), cuda(np.array([3, 1, 4, 0], np.int32)), torch.arange(40, **i32)
    count, same = torch.full((1,), 9, **i32), torch.full((2, 2), 20, **i32)
    parents = cuda(np.array([[0, 0], [1, 1]], np.int32))  # (the same again changes nothing more)
    calls = {
        "kv_pages": lambda s: own.kv_pages(lengths, new, tables.clone() if s is None else tables, free, count, 16, 12, stream=s),
        "kv_store": lambda s: (own.kv_store(cache, x[:, 4:6], x[:, 6:], slots, x[:, :4], positions, freqs, stream=s),),
        "kv_attention": lambda s: (own.kv_attention(cache, x[:, :4], tables, positions, stream=s),),
        "beam_select": lambda s: own.beam_select(logits, scores, 4, stream=s),
        "beam_reorder": lambda s: own.beam_reorder(parents, same, tables, [cache], stream=s) or (),
    }
    call = calls[name]
    want = call(None)
    own.sync()
    s = torch.cuda.Stream()
    at = s.cuda_stream if handle else s
    torch.cuda.synchronize()
    call(at)
    big = torch.ones((8192, 8192), device="cuda")
    out = torch.mm(big, big)
    torch.cuda.synchronize()
    sizes = [k * 512 for k in (1, 2, 4, 8, 16, 24)] + [t.numel() * t.element_size() for t in want]
    taken = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(64)]
    torch.cuda.synchronize()
    for _ in range(20):
        torch.mm(big, big, out=out)
    for t in taken:
        t.fill_(7)
    del t
    taken = taken[::2]
    got = call(at)
    s.synchronize()
    busy = not torch.cuda.current_stream().query()
    torch.cuda.synchronize()
    assert busy
    own.sync()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    own.close()


def test_python_checks(ctx):
    cache = rlq.KvCache.make(DT.F16, 4, 2, 16, 64)
    q, t = torch.zeros((2, 4, 64), device="cuda"), torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ctx.kv_attention(cache, q[:, :, :32], t, pos)
    with pytest.raises(TypeError):
        ctx.kv_attention(cache, q.transpose(1, 2).contiguous().transpose(1, 2), t, pos)
    with pytest.raises(TypeError):
        ctx.kv_attention(cache, q[:1].expand(2, 4, 64), t, pos)
    with pytest.raises(TypeError):
        ctx.kv_attention(cache, q.cpu(), t, pos)
    with pytest.raises(TypeError):
        ctx.kv_attention(cache, q, t.long(), pos)
    with pytest.raises(ValueError):
        ctx.kv_attention(cache, q, t, pos[:1])
    with pytest.raises(TypeError):
        rlq.KvCache(cache.k.float(), cache.v, DT.F16, 16, 64)
    with pytest.raises(ValueError):
        rlq.KvCache(cache.k, cache.v, DT.F16, 32, 32)
    with raises("Shape", 3, 2):
        ctx.kv_attention(cache, q[:, :3], t, pos)
    with raises("Unimplemented"):
        rlq.KvCache.make(DT.Q4_K, 1, 1, 16, 64)
