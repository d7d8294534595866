"""rlq_rms_norm against the oracle: the residual's addition in numpy's f32, the
norm by the reference's sequential arithmetic and its blocks by the reference's
quantizers, all bit for bit.  Shapes cross the kernel's variants (64, 256 and 1024
lanes a row, one to eight units of four values a lane, rows without 16-byte alignment)."""
import numpy as np
import pytest

import oracle as O
from rlq_loader import load

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType
EPS = 1e-5


def say(*a):
    print("[case]", *a, flush=True)


@pytest.fixture(scope="module")
def ctx():
    c = rlq.Context(0)
    yield c
    c.close()


def rows_of(seed, rows, cols, loud=True):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    if loud:
        x[:, rng.random(cols) < 0.02] *= np.float32(30.0)
    return x


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


def check(total, y, q, x, residual, w, packed, eps=EPS, rows=None):
    t = x if residual is None else x + residual
    for r in range(x.shape[0]) if rows is None else rows:
        want = O.rms_norm(t[r], w, eps)
        if total is not None:
            assert np.array_equal(bits(total[r].cpu().numpy()), bits(t[r])), r
        if y is not None:
            assert np.array_equal(bits(y[r].cpu().numpy()), bits(want)), r
        if q is not None:
            assert np.array_equal(q[r].cpu().numpy(), O.quantize(int(packed), want)), r


SHAPES = [(1, 256), (2, 256), (17, 256), (16, 512), (5, 1024), (1, 1280), (1, 4096), (33, 4096), (3, 4352), (2, 8192),
          (2, 8448), (3, 16384), (2, 16640), (1, 32768), (300, 768)]


@pytest.mark.parametrize("packed", [None, DT.Q8_K, DT.Q8_0], ids=lambda p: p.name if p is not None else "f32")
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rows(ctx, rows, cols, packed):
    say("norm", rows, cols, packed)
    x, res, w = rows_of(1, rows, cols), rows_of(2, rows, cols), rows_of(3, 1, cols, False)[0]
    total, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, residual=gpu(res), packed=packed)
    ctx.sync()
    check(total, y, q, x, res, w, packed)
    total, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, packed=packed)
    ctx.sync()
    assert total is None
    check(None, y, q, x, None, w, packed)


@pytest.mark.parametrize("rows,cols", [(1, 32), (40, 32), (3, 96), (333, 896), (2, 1056), (1, 14336 + 32), (1, 32736)])
def test_rows_of_half_blocks(ctx, rows, cols):
    """Q8_0 rows that are no whole number of 256 values."""
    say("norm Q8_0", rows, cols)
    x, res, w = rows_of(4, rows, cols), rows_of(5, rows, cols), rows_of(6, 1, cols, False)[0]
    total, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, residual=gpu(res), packed=DT.Q8_0)
    ctx.sync()
    check(total, y, q, x, res, w, DT.Q8_0)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (20, 17), (2, 100), (7, 255), (3, 1023), (2, 4095), (2, 5001),
                                       (1, 20001), (1, 32767), (9, 36)])
def test_any_length(ctx, rows, cols):
    say("norm f32", rows, cols)
    x, res, w = rows_of(7, rows, cols), rows_of(8, rows, cols), rows_of(9, 1, cols, False)[0]
    total, y, _ = ctx.rms_norm(gpu(x), gpu(w), EPS, residual=gpu(res))
    ctx.sync()
    check(total, y, None, x, res, w, None)


@pytest.mark.parametrize("cols,packed", [(512, DT.Q8_K), (4096, DT.Q8_K), (896, DT.Q8_0), (100, None)])
def test_unaligned_views(ctx, cols, packed):
    say("norm unaligned", cols, packed)
    rows = 3
    x, w = rows_of(10, rows, cols), rows_of(11, 1, cols, False)[0]
    xs = torch.zeros(rows * cols + 1, device="cuda")[1:].view(rows, cols)
    ws = torch.zeros(cols + 3, device="cuda")[3:]
    out = torch.zeros(rows * cols + 1, device="cuda")[1:].view(rows, cols)
    xs.copy_(gpu(x)), ws.copy_(gpu(w))
    _, y, q = ctx.rms_norm(xs, ws, EPS, packed=packed, y=out)
    ctx.sync()
    check(None, y, q, x, None, w, packed)


@pytest.mark.parametrize("cols", [64, 256, 1024, 4096, 16384])
def test_mean_between_two_floats(ctx, cols):
    """A sum of squares whose mean lies halfway between two f32 values: the kernel's
    parallel sum cannot tell the reference's rounding and repeats it in order."""
    say("norm halfway", cols)
    root = np.float32(np.sqrt(cols))
    for small in (2.0 ** -12, 2.0 ** -12 * (1 + 2.0 ** -20), 2.0 ** -12 * (1 - 2.0 ** -20)):
        x = np.zeros((3, cols), np.float32)
        x[0, 0], x[0, cols - 1] = root, root * np.float32(small)
        x[1, cols - 1], x[1, 0] = root, root * np.float32(small)
        x[2] = rows_of(12, 1, cols)[0]
        w = np.ones(cols, np.float32)
        _, y, _ = ctx.rms_norm(gpu(x), gpu(w), EPS)
        ctx.sync()
        check(None, y, None, x, None, w, None)


@pytest.mark.parametrize("cols", [256, 1024, 4096, 8192, 32768])
def test_in_place(ctx, cols):
    say("norm in place", cols)
    rows = 5
    x, res, w = rows_of(13, rows, cols), rows_of(14, rows, cols), rows_of(15, 1, cols, False)[0]
    xs, rs = gpu(x), gpu(res)
    total, y, q = ctx.rms_norm(xs, gpu(w), EPS, residual=rs, packed=DT.Q8_K, total=rs, y=xs)
    ctx.sync()
    assert total is rs and y is xs
    check(total, y, q, x, res, w, DT.Q8_K)


def test_outputs_on_their_own(ctx):
    say("norm outputs")
    x, res, w = rows_of(16, 4, 512), rows_of(17, 4, 512), rows_of(18, 1, 512, False)[0]
    total, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, packed=DT.Q8_0, normed=False)
    assert total is None and y is None
    check(None, None, q, x, None, w, DT.Q8_0)
    given = torch.empty((4, 512), device="cuda")
    total, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, total=given)
    check(total, y, None, x, None, w, None)
    x3 = gpu(x).view(2, 2, 512)
    _, y, q = ctx.rms_norm(x3, gpu(w), EPS, packed=DT.Q8_K)
    ctx.sync()
    assert y.shape == (2, 2, 512) and q.shape == (4, rlq.row_bytes(DT.Q8_K, 512))
    check(None, y.view(4, 512), q, x, None, w, DT.Q8_K)


def test_shapes_refused(ctx):
    x, w = torch.zeros((2, 256), device="cuda"), torch.ones(256, device="cuda")
    for kw in (dict(residual=torch.zeros((1, 256), device="cuda")), dict(y=torch.zeros((3, 256), device="cuda")),
               dict(total=torch.zeros(1, device="cuda")), dict(q=torch.zeros(10, dtype=torch.uint8, device="cuda")),
               dict(packed=DT.Q8_K, q=torch.zeros(10, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            ctx.rms_norm(x, w, EPS, **kw)
    with pytest.raises(ValueError):
        ctx.rms_norm(x, torch.ones(255, device="cuda"), EPS)
    with pytest.raises(TypeError):
        ctx.rms_norm(x.half(), w, EPS)
    with pytest.raises(TypeError):
        ctx.rms_norm(x.t().contiguous().t(), torch.ones(256, device="cuda"), EPS)
    total, y, q = ctx.rms_norm(x[:0], w, EPS, packed=DT.Q8_K)
    assert y.shape == (0, 256) and q.shape[0] == 0


@pytest.mark.parametrize("cols", [256, 1024, 4096, 16384, 32768])
@pytest.mark.parametrize("what", ["nan", "inf", "overflow", "weight", "scale"])
def test_bad_row_is_held_back(ctx, cols, what):
    """A row with a data error keeps its old outputs, the others are written."""
    say("norm bad", cols, what)
    rows, at, bad = 7, cols - 3, 5
    x, w = rows_of(19, rows, cols), np.ones(cols, np.float32)
    code, a = "NonFinite", 2
    if what == "nan":
        x[bad, at], a = np.nan, 1  # the squares' sum, and so the scale, is NaN
    elif what == "inf":
        x[bad, at], a = np.inf, 1  # the scale is 0
    elif what == "overflow":
        x[bad, at], a = 3e38, 1  # the square is infinite
    elif what == "weight":
        x[:, at] = 0.0
        x[bad, at], w[at] = 1.0, np.inf
        x[np.arange(rows) != bad, at] = 1.0
        bad = None  # every row is refused: 1 * scale * inf
    else:  # a block whose levels have no finite scale
        x[bad, :256], code, a = 1e-38, "UnrepresentableScale", 0
        x[bad, 256:] = 0.0
    total = torch.full((rows, cols), 7.0, device="cuda")
    y = torch.full((rows, cols), 7.0, device="cuda")
    q = torch.full((rows, rlq.row_bytes(DT.Q8_K, cols)), 77, dtype=torch.uint8, device="cuda")
    eps = EPS if what != "scale" else 1.0
    ctx.rms_norm(gpu(x), gpu(w), eps, packed=DT.Q8_K, total=total, y=y, q=q)
    with pytest.raises(rlq.QuantError) as e:
        ctx.sync()
    assert (e.value.name, e.value.a, e.value.b) == (code, a, bad or 0)
    ctx.sync()  # cleared
    held = range(rows) if bad is None else [bad]
    for r in held:
        assert bool((total[r] == 7.0).all()) and bool((y[r] == 7.0).all()) and bool((q[r] == 77).all()), r
    check(total, y, q, x, None, w, DT.Q8_K, eps, [r for r in range(rows) if r not in held])


def test_zero_rows_and_lowest_values(ctx):
    """Rows of zeros (a block of scale 0) and of the largest values whose squares
    are finite."""
    say("norm zeros")
    x = np.zeros((3, 512), np.float32)
    x[1] = np.float32(1.5e19)
    x[2, ::7] = np.float32(-1.8e19)
    w = np.full(512, 0.5, np.float32)
    _, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, packed=DT.Q8_K)
    ctx.sync()
    check(None, y, q, x, None, w, DT.Q8_K)


def test_packed_rows_feed_the_products(ctx):
    """The packed output is a right-hand side of mul_mat: the products of the
    quantized rows bit for bit."""
    say("norm to mul_mat")
    from test_gpu_sweep import _weights
    rows, cols, n = 48, 1024, 3
    W = rlq.Weights(ctx, DT.Q6_K, _weights(DT.Q6_K, rows, cols, 5), rows, cols)
    x, w = rows_of(20, n, cols), rows_of(21, 1, cols, False)[0]
    _, y, q = ctx.rms_norm(gpu(x), gpu(w), EPS, packed=DT.Q8_K)
    got = ctx.mul_mat(W, q.view(1, 1, n, -1), x_dtype=DT.Q8_K)
    want = ctx.mul_mat(W, ctx.quantize(DT.Q8_K, y).view(1, 1, n, -1), x_dtype=DT.Q8_K)
    ctx.sync()
    assert torch.equal(got, want)
    W.close()


def test_replayed(ctx):
    say("norm replayed")
    x, w = rows_of(22, 6, 4096), rows_of(23, 1, 4096, False)[0]
    xs, ws, y, q = gpu(x), gpu(w), torch.empty((6, 4096), device="cuda"), torch.empty(
        (6, rlq.row_bytes(DT.Q8_K, 4096)), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ctx.rms_norm(xs, ws, EPS, packed=DT.Q8_K, y=y, q=q)
    for k in range(4):
        x = rows_of(30 + k, 6, 4096)
        xs.copy_(gpu(x))
        y.zero_(), q.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(None, y, q, x, None, w, DT.Q8_K)
        ctx.rms_norm(gpu(x), ws, EPS)
    ctx.sync()
