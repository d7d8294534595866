"""Beam search on the GPU (rlq_beam_select, rlq_beam_reorder) against plain 64-bit
forms, and beams decoded over a paged cache against sequences that share nothing."""
import numpy as np
import pytest

import kv_oracle as K
from rlq_loader import load
from test_gpu_kv import Pages, cuda, fill, raises, say

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType


@pytest.fixture(scope="module")
def ctx():
    c = rlq.Context(0)
    yield c
    c.close()


def check(got, want):
    scores, parents, tokens = (t.cpu().numpy() for t in got)
    assert np.array_equal(parents, want[1]) and np.array_equal(tokens, want[2])
    some = want[1] >= 0
    assert (scores[~some] == -np.inf).all()
    # one rounding to f32, and the sum's exponentials: each within 2^-22, so the log's argument too
    assert (np.abs(scores[some] - want[0][some]) <= 2.0 ** -24 * np.abs(want[0][some]) + 2.0 ** -22).all()


def choose(ctx, z, scores, best):
    got = ctx.beam_select(cuda(z), cuda(scores), best)
    ctx.sync()
    check(got, K.select(z, scores, best))
    return got


@pytest.mark.parametrize("vocabulary", [1, 2, 63, 64, 65, 255, 257, 1000, 4095, 4096, 4097, 8193, 32000, 50257])
@pytest.mark.parametrize("beams", [1, 4, 7])
def test_select(ctx, vocabulary, beams):
    rng = np.random.default_rng(vocabulary + beams)
    for groups, best in ((1, 1), (3, 2 * beams), (2, 33)):
        best = min(best, beams * vocabulary)
        say("select", groups, beams, vocabulary, best)
        z = (rng.standard_normal((groups, beams, vocabulary)) * 3).astype(np.float32)
        z[rng.random(z.shape) < 0.05] = -np.inf
        scores = (-10 * rng.random((groups, beams))).astype(np.float32)
        scores[rng.random(scores.shape) < 0.2] = -np.inf
        choose(ctx, z, scores, best)


@pytest.mark.parametrize("groups,beams,vocabulary,best", [(1, 64, 3000, 64), (2, 16, 151936, 32), (40, 3, 9001, 64), (300, 2, 700, 4),
                                                          (1, 1, 200000, 64), (5, 33, 1025, 17)])
def test_select_large(ctx, groups, beams, vocabulary, best):
    say("select", groups, beams, vocabulary, best)
    rng = np.random.default_rng(best)
    z = (rng.standard_normal((groups, beams, vocabulary)) * 4).astype(np.float32)
    choose(ctx, z, (-3 * rng.random((groups, beams))).astype(np.float32), best)


def test_select_equal_logits(ctx):
    """Ties go to the lowest beam and token: everywhere equal, many equal ones at the border, equal beams."""
    rng = np.random.default_rng(1)
    for vocabulary in (64, 5000, 20000):
        say("select ties", vocabulary)
        choose(ctx, np.zeros((2, 3, vocabulary), np.float32), np.zeros((2, 3), np.float32), 40)
        z = rng.integers(-3, 4, (2, 4, vocabulary)).astype(np.float32)
        z[:, 1] = z[:, 0]
        choose(ctx, z, np.zeros((2, 4), np.float32), 64)
        z = np.where(rng.random((1, 2, vocabulary)) < 0.5, 0.0, -0.0).astype(np.float32)
        choose(ctx, z, np.zeros((1, 2), np.float32), 20)
    z = np.sort(rng.standard_normal((1, 2, 30000)).astype(np.float32))  # the best at a row's end, then at its start
    choose(ctx, z, np.zeros((1, 2), np.float32), 64)
    choose(ctx, np.ascontiguousarray(z[..., ::-1]), np.zeros((1, 2), np.float32), 64)


def test_select_far_logits(ctx):
    """Logits of the type's ends, few that may follow, one that takes all."""
    say("select far")
    low = np.finfo(np.float32).min
    z = np.full((3, 2, 6000), low, np.float32)
    z[0, 0, 17], z[0, 1, 5999] = 5, 7
    z[1] = -np.inf
    z[1, 0, 3], z[1, 1, 4] = 1, -np.float32(3e38)
    z[2, 0] = -np.inf
    z[2, 1, :] = -1e30
    choose(ctx, z, np.array([[-1, -2], [0, 0], [0, -5]], np.float32), 6)
    got = choose(ctx, np.full((2, 2, 300), -np.inf, np.float32), np.zeros((2, 2), np.float32), 3)
    assert (got[1] == -1).all()
    choose(ctx, z, np.full((3, 2), -np.inf, np.float32), 3)


@pytest.mark.parametrize("beams,vocabulary,best", [(1, 20000, 4), (3, 20000, 4), (3, 20000, 40), (32, 20000, 8), (32, 20000, 16), (2, 300, 8)])
def test_select_scores_that_hide_the_logits(ctx, beams, vocabulary, best):
    """Beside the type's lowest score every logit is rounded away: ranks are equal, a beam's order is that of its logits."""
    say("select hidden", beams, vocabulary, best)
    rng = np.random.default_rng(best)
    z = rng.standard_normal((2, beams, vocabulary)).astype(np.float32)
    scores = np.full((2, beams), np.finfo(np.float32).min, np.float32)
    z[1, 0, np.arange(vocabulary) != 7] = -np.inf  # a live beam of one token before them
    scores[1, 0] = 0
    got = ctx.beam_select(cuda(z), cuda(scores), best)
    ctx.sync()
    for g in range(2):
        want = [(0, 7)] if g else []
        for b in range(g, beams):
            want += [(b, t) for t in np.argsort(-z[g, b], kind="stable")[:best]]
        want += [(-1, -1)] * best
        assert [(int(p), int(t)) for p, t in zip(got[1][g].tolist(), got[2][g].tolist())] == [(b, int(t)) for b, t in want[:best]]


def test_select_errors_are_the_groups_own(ctx):
    say("select errors")
    rng = np.random.default_rng(2)
    z = rng.standard_normal((4, 3, 9000)).astype(np.float32)
    scores = rng.standard_normal((4, 3)).astype(np.float32)
    want = K.select(z, scores, 5)
    for where, value in (((2, 1, 8999), np.nan), ((2, 0, 0), np.inf), ((2, 2, 4321), -np.nan), (None, np.nan), (None, np.inf)):
        y, s = z.copy(), scores.copy()
        if where:
            y[where] = value
        else:
            s[2, 1] = value
        got = ctx.beam_select(cuda(y), cuda(s), 5)
        with raises("NonFinite", 4, 2):
            ctx.sync()
        others = [0, 1, 3]
        check([t[others] for t in got], [w[others] for w in want])
        assert (got[0][2] == -np.inf).all() and (got[1][2] == -1).all() and (got[2][2] == -1).all()
        if where:  # a beam without a place is not looked at
            s[2, where[1]] = -np.inf
            choose(ctx, np.where(np.isfinite(y), y, 0).astype(np.float32), s, 5)
            got = ctx.beam_select(cuda(y), cuda(s), 5)
            ctx.sync()
            check(got, K.select(np.where(np.isfinite(y), y, 0), s, 5))


def test_select_strides_streams_and_replays(ctx):
    say("select strides")
    rng = np.random.default_rng(3)
    z = rng.standard_normal((3, 4, 8000)).astype(np.float32)
    scores = rng.standard_normal((3, 4)).astype(np.float32)
    want = ctx.beam_select(cuda(z), cuda(scores), 8)
    wide = torch.full((3, 4, 8003), float("nan"), device="cuda")
    wide[..., 1:8001] = cuda(z)
    for part in (wide[..., 1:8001],):
        for a, b in zip(ctx.beam_select(part, cuda(scores), 8), want):
            assert torch.equal(a, b)
    with pytest.raises(TypeError):
        ctx.beam_select(wide[:, ::2, 1:8001].transpose(0, 1), cuda(scores)[:, ::2].t().contiguous(), 8)
    s = torch.cuda.Stream()
    zc, sc = cuda(z), cuda(scores)
    torch.cuda.synchronize()
    for a, b in zip(ctx.beam_select(zc, sc, 8, stream=s), want):
        s.synchronize()
        assert torch.equal(a, b)
    out = tuple(torch.zeros_like(t) for t in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.beam_select(zc, sc, 8, out=out)
    for k in range(4):
        for t in out:
            t.zero_()
        graph.replay()
        choose(ctx, z[:1, :2, :100 * (k + 1)].copy(), scores[:1, :2].copy(), 3)
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    ctx.sync()


# ---- reorder ----------------------------------------------------------------------------


def reorder(ctx, rng, dtype, groups, beams, layers, kv, dim, page, lengths, parents=None):
    width = max(lengths) // page + 2
    pool = groups * beams * width + 3
    caches = [rlq.KvCache.make(dtype, pool, kv, page, dim) for _ in range(layers)]
    for c in caches:
        fill(rng, c)
    tables = rng.permutation(pool)[:groups * beams * width].astype(np.int32).reshape(groups * beams, width)
    if parents is None:
        parents = rng.integers(-1, beams, (groups, beams)).astype(np.int32)
    size = np.repeat(np.asarray(lengths, np.int32), beams).reshape(groups, beams)
    want_t = tables.copy()
    before = [[t.cpu().numpy().copy() if dtype != DT.BF16 else t.cpu().view(torch.int16).numpy().copy() for t in (c.k, c.v)]
              for c in caches]
    want = [[t.copy() for t in c] for c in before]
    for g in range(groups):
        n, rows = size[g, 0] // page, size[g, 0] % page
        for b in range(beams):
            p = parents[g, b]
            if p < 0:
                continue
            i, j = g * beams + b, g * beams + p
            want_t[i, :n] = tables[j, :n]
            for a, w in zip(before, want):
                for x, y in zip(a, w):
                    if not rows:
                        continue
                    if dtype == DT.Q8_0:
                        for lo, per in ((0, dim), (page * dim, dim // 16)):
                            y[tables[i, n], :, lo:lo + rows * per] = x[tables[j, n], :, lo:lo + rows * per]
                    else:
                        y[tables[i, n], :, :rows] = x[tables[j, n], :, :rows]
    t = cuda(tables)
    ctx.beam_reorder(cuda(parents), cuda(size), t, caches)
    ctx.sync()
    assert np.array_equal(t.cpu().numpy(), want_t)
    for c, w in zip(caches, want):
        for x, y in zip((c.k, c.v), w):
            assert np.array_equal((x if dtype != DT.BF16 else x.view(torch.int16)).cpu().numpy(), y)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F16, DT.BF16, DT.Q8_0])
@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 16, 17, 32])
def test_reorder(ctx, dtype, beams):
    rng = np.random.default_rng(beams)
    for kv, dim, page, lengths in ((2, 64, 16, [37, 0, 48]), (1, 32, 64, [1, 63]), (3, 96, 32, [31, 64, 5])):
        say("reorder", dtype, beams, kv, dim, page)
        reorder(ctx, rng, dtype, len(lengths), beams, 2, kv, dim, page, lengths)


def test_reorder_changes_places(ctx):
    """Beams in a ring, swapped, all from one, none."""
    rng = np.random.default_rng(1)
    for parents in ([[1, 2, 3, 0]], [[1, 0, 3, 2]], [[3, 3, 3, 3]], [[0, 1, 2, 3]], [[-1, -1, 0, -1]]):
        say("reorder places", parents)
        reorder(ctx, rng, DT.F16, 1, 4, 3, 2, 64, 16, [75], np.array(parents, np.int32))


def test_reorder_of_many_layers(ctx):
    for layers in (64, 65, 130):
        say("reorder layers", layers)
        reorder(ctx, np.random.default_rng(layers), DT.BF16, 2, 3, layers, 1, 32, 16, [23, 30])


def test_reorder_errors_are_the_groups_own(ctx):
    say("reorder errors")
    cache = rlq.KvCache.make(DT.F16, 12, 1, 16, 32)
    fill(np.random.default_rng(1), cache)
    for change, a in ((lambda p, n, t: p.__setitem__((1, 1), 2), 3), (lambda p, n, t: p.__setitem__((1, 0), -2), 2),
                      (lambda p, n, t: n.__setitem__((1, 1), 21), 3), (lambda p, n, t: n.__setitem__((1, slice(None)), -1), 2),
                      (lambda p, n, t: n.__setitem__((1, slice(None)), 33), 2), (lambda p, n, t: t.__setitem__((3, 1), 12), 3),
                      (lambda p, n, t: t.__setitem__((2, 1), -1), 2)):
        parents, lengths = np.array([[1, 0], [1, 0], [1, 1]], np.int32), np.full((3, 2), 20, np.int32)
        tables = np.arange(12, dtype=np.int32).reshape(6, 2)
        change(parents, lengths, tables)
        mine = rlq.KvCache(cache.k.clone(), cache.v.clone(), DT.F16, 16, 32)
        t = cuda(tables)
        ctx.beam_reorder(cuda(parents), cuda(lengths), t, [mine])
        with raises("Bounds", a):
            ctx.sync()
        got = t.cpu().numpy()
        assert np.array_equal(got[2:4], tables[2:4]) and got[:2, 0].tolist() == [2, 0] and got[4:, 0].tolist() == [10, 10]
        assert torch.equal(mine.k[4:8], cache.k[4:8]) and torch.equal(mine.v[4:8], cache.v[4:8])
        assert torch.equal(mine.k[1, :, :4], cache.k[3, :, :4]) and torch.equal(mine.k[1, :, 4:], cache.k[1, :, 4:])


def test_beams_decoded_together(ctx):
    """A prompt, then beams of two groups over 50 steps with every call of a step, against
    sequences stored whole and on their own: the same keys and values in the same
    places, so the same attention bit for bit."""
    say("beams together")
    rng = np.random.default_rng(5)
    groups, beams, heads, kv, dim, page, vocabulary, width = 2, 3, 4, 2, 64, 16, 500, 8
    n, prompt = groups * beams, 21
    p = Pages(n, width, n * width, page, 6, owned=True)
    caches = [rlq.KvCache.make(DT.F16, p.pages, kv, page, dim) for _ in range(2)]
    tables = p.on["tables"]
    keys = [[[] for _ in range(n)] for _ in caches]  # each beam's whole history
    head = cuda(rng.standard_normal((heads * dim, vocabulary)).astype(np.float32))
    embed = rng.standard_normal((2, vocabulary, (heads + 2 * kv) * dim)).astype(np.float32)
    freqs = cuda((10000.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32))

    def layer(i, tokens, row_beams, slots, positions, requests):
        x = cuda(embed[i][tokens])
        k, v = (x[:, a * dim:b * dim].unflatten(1, (kv, dim)) for a, b in ((heads, heads + kv), (heads + kv, heads + 2 * kv)))
        q = ctx.kv_store(caches[i], k, v, slots, x[:, :heads * dim].unflatten(1, (heads, dim)), positions, freqs)
        for t, b in enumerate(row_beams):
            keys[i][b].append((k[t].clone(), v[t].clone()))
        y = ctx.kv_attention(caches[i], q, tables, positions, requests)
        for t, b in enumerate(row_beams):  # the beam alone, in a cache of its own
            if t % 5 and len(row_beams) > n:
                continue
            have = len(keys[i][b]) if len(row_beams) <= n else int(positions[t]) + 1
            own = rlq.KvCache.make(DT.F16, width, kv, page, dim)
            ks, vs = (torch.stack([e[j] for e in keys[i][b][:have]]) for j in range(2))
            at = torch.arange(have, device="cuda")
            ctx.kv_store(own, ks, vs, at, torch.zeros((have, heads, dim), device="cuda"), at.int(), freqs)
            one = ctx.kv_attention(own, q[t:t + 1].contiguous(), torch.arange(width, device="cuda").int().view(1, -1),
                                   cuda(np.array([have - 1], np.int32)))
            assert torch.equal(one[0], y[t])
        return y

    # the groups' first beams take the prompt; the others only the page that it leaves part-filled
    new = np.zeros(n, np.int32)
    new[::beams] = prompt
    _, _, _, slots, positions, requests = p.step(ctx, new, int(new.sum()))
    tokens = rng.integers(0, vocabulary, int(new.sum()))
    row_beams = requests.cpu().numpy()
    for i in range(2):
        layer(i, tokens, row_beams, slots, positions, requests)
    p.lengths = np.where(new > 0, p.lengths, prompt // page * page).astype(np.int32)
    p.on["lengths"] = cuda(p.lengths)
    p.step(ctx, np.where(new > 0, 0, prompt % page), n * page)
    assert (p.lengths == prompt).all()
    parents = torch.zeros((groups, beams), dtype=torch.int32, device="cuda")
    scores = torch.tensor([[0.0] + [-float("inf")] * (beams - 1)] * groups, device="cuda")
    tokens = rng.integers(0, vocabulary, n)
    for step in range(50):
        ctx.beam_reorder(parents, p.on["lengths"].view(groups, beams), tables, caches)
        ctx.sync()
        p.tables[:] = tables.cpu().numpy()
        source = (parents.cpu().numpy() + np.arange(0, n, beams)[:, None]).reshape(-1)
        for i in range(2):
            keys[i] = [list(keys[i][s]) for s in source]
        _, _, _, slots, positions, requests = p.step(ctx, np.ones(n), n)
        y = [layer(i, tokens, np.arange(n), slots, positions, requests) for i in range(2)][1]
        logits = (y.reshape(n, -1) @ head).view(groups, beams, vocabulary)
        old = scores
        scores, parents, token = ctx.beam_select(logits, scores, beams)
        ctx.sync()
        check((scores, parents, token), K.select(logits.cpu().numpy(), old.cpu().numpy(), beams))
        tokens = token.view(-1).cpu().numpy()
    p.step(ctx, np.full(n, -1), 0)
    assert p.count[0] == p.pages and sorted(p.free) == list(range(p.pages))
