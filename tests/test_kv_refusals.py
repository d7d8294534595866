"""Refusals of the paged-cache and beam entry points, which come before any device
work: no GPU is needed.  The context is a stand-in; no pointer is followed on these paths."""
import ctypes

import pytest

from rlq_loader import load
from test_moe_refusals import CTX, P, call, check

rlq = load()
NAMES = {v: k for k, v in rlq.ERROR_NAMES.items()}
F32, F16, Q8_0, Q4_K, BF16 = 0, 1, 8, 12, 30
REF = ctypes.byref(CTX)


def cache(k=P, v=2 * P, dtype=F16, kv_heads=2, page=16, dim=64, pages=5, k_stride=4096, v_stride=4096):
    return rlq._KvCacheT(k, v, dtype, kv_heads, page, dim, pages, k_stride, v_stride)


def ref(c):
    return None if c is None else ctypes.byref(c)


def pages(ctx=REF, before=P, more=P, requests=3, page=16, tables=P, owned=None, width=4, free=P, count=P, n=12, tokens=5,
          after=P, count_after=P, starts=P, slots=P, positions=P, out=P):
    return call("rlq_kv_pages", ctx, before, more, requests, page, tables, owned, width, free, count, n, tokens, after,
                count_after, starts, slots, positions, out, None)


def test_pages():
    check(pages(ctx=None), "InvalidArgument")
    for k in ("before", "more", "tables", "free", "count", "after", "count_after", "starts", "slots", "positions", "out"):
        check(pages(**{k: None}), "InvalidArgument")
        check(pages(**{k: P + 2}), "InvalidArgument")
    check(pages(owned=P + 1), "InvalidArgument")
    check(pages(slots=P + 4), "InvalidArgument")
    for page in (0, 1, 8, 15, 17, 48, 512, 2 ** 40):
        check(pages(page=page), "Unimplemented", page, 256)
    check(pages(requests=0), "InvalidMatrixShape", 0, 4)
    check(pages(requests=4097), "Unimplemented", 4097, 4096)
    for k in ("width", "n", "tokens"):
        check(pages(**{k: 2 ** 31}), "Unimplemented", 2 ** 31, 2 ** 31 - 1)


BAD_CACHES = [
    (dict(k=None), "InvalidArgument", 0, 0), (dict(v=None), "InvalidArgument", 0, 0), (dict(k=P + 8), "InvalidArgument", 0, 0),
    (dict(v=P), "InvalidArgument", 0, 0), (dict(dtype=99), "InvalidType", 0, 0), (dict(dtype=Q4_K), "Unimplemented", 0, 0),
    (dict(page=24), "Unimplemented", 24, 256), (dict(page=0), "Unimplemented", 0, 256), (dict(dim=80), "NonMultiple", 80, 32),
    (dict(dim=0), "NonMultiple", 0, 32), (dict(dim=288), "Unimplemented", 288, 256),
    (dict(kv_heads=0), "InvalidMatrixShape", 5, 0), (dict(pages=0), "InvalidMatrixShape", 0, 2),
    (dict(kv_heads=65536, k_stride=2 ** 40, v_stride=2 ** 40), "Unimplemented", 65536, 65535),
    (dict(pages=2 ** 31), "Unimplemented", 2 ** 31, 2 ** 31 - 1), (dict(k_stride=4080), "InvalidLength", 4096, 4080),
    (dict(v_stride=4095), "InvalidLength", 4096, 4095), (dict(v_stride=4104), "NonMultiple", 4104, 16),
    (dict(k_stride=2 ** 62), "SizeOverflow", 0, 0), (dict(dtype=F32), "InvalidLength", 8192, 4096),
    (dict(dtype=Q8_0, k_stride=2160), "InvalidLength", 2176, 2160)]


def store(ctx=REF, c=None, null_cache=False, q=P, q_stride=512, heads=4, k=P, k_stride=512, v=P, v_stride=512, tokens=3, slots=P,
          positions=P, freqs=P, half=32, flags=1, q_out=P, out_stride=512):
    c = None if null_cache else c or cache()
    return call("rlq_kv_store", ctx, ref(c), q, q_stride, heads, k, k_stride, v, v_stride, tokens, slots, positions, freqs, half,
                flags, q_out, out_stride, None)


def attend(ctx=REF, c=None, null_cache=False, q=P, q_stride=512, rows=3, heads=4, tables=P, table_rows=3, width=4, positions=P,
           requests=P, scale=0.0, window=0, out=P, out_stride=512):
    c = None if null_cache else c or cache()
    return call("rlq_kv_attention", ctx, ref(c), q, q_stride, rows, heads, tables, table_rows, width, positions, requests, scale,
                window, out, out_stride, None)


def reorder(ctx=REF, caches=None, null_cache=False, parents=P, lengths=P, groups=2, beams=4, tables=P, width=4, n=None):
    caches = caches or [cache(), cache()]
    layers = (rlq._KvCacheT * len(caches))(*caches)
    return call("rlq_beam_reorder", ctx, parents, lengths, groups, beams, tables, width, None if null_cache else layers,
                len(caches) if n is None else n, None)


@pytest.mark.parametrize("change,name,a,b", BAD_CACHES)
def test_caches(change, name, a, b):
    c = cache(**change)
    check(store(c=c), name, a, b)
    check(attend(c=c), name, a, b)
    check(reorder(caches=[cache(), c] if name != "Unimplemented" or a == 0 else [c]), name, a, b)


def test_store():
    check(store(ctx=None), "InvalidArgument")
    check(store(null_cache=True), "InvalidArgument")
    check(store(flags=2), "InvalidArgument", 2)
    for k in ("q", "k", "v", "slots", "positions", "freqs", "q_out"):
        check(store(**{k: None}), "InvalidArgument")
        check(store(**{k: P + 2}), "InvalidArgument")
    check(store(slots=P + 4), "InvalidArgument")
    check(store(half=33), "Shape", 33, 32)
    check(store(heads=65536), "Unimplemented", 65536, 65535)
    check(store(k_stride=127), "InvalidLength", 128, 127)
    check(store(v_stride=127), "InvalidLength", 128, 127)
    check(store(q_stride=255), "InvalidLength", 256, 255)
    check(store(out_stride=255), "InvalidLength", 256, 255)
    check(store(out_stride=520), "InvalidArgument")  # in place, but elsewhere
    check(store(tokens=8388607), "Unimplemented", 8388607, 8388606)
    check(store(tokens=0, k=None, v=None, slots=None, q=None), None)


def test_attention():
    check(attend(ctx=None), "InvalidArgument")
    check(attend(null_cache=True), "InvalidArgument")
    for k in ("q", "tables", "positions", "out"):
        check(attend(**{k: None}), "InvalidArgument")
        check(attend(**{k: P + 2}), "InvalidArgument")
    check(attend(requests=P + 2), "InvalidArgument")
    check(attend(heads=0), "Shape", 0, 2)
    check(attend(heads=5), "Shape", 5, 2)
    check(attend(heads=65536), "Unimplemented", 65536, 65535)
    for scale in (float("nan"), float("inf"), -float("inf")):
        check(attend(scale=scale), "InvalidConfig", 6)
    check(attend(rows=65536), "Unimplemented", 65536, 65535)
    for k in ("table_rows", "width", "window"):
        check(attend(**{k: 2 ** 31}), "Unimplemented", 2 ** 31, 2 ** 31 - 1)
    check(attend(q_stride=255), "InvalidLength", 256, 255)
    check(attend(out_stride=255), "InvalidLength", 256, 255)
    check(attend(requests=None, table_rows=2), "Shape", 2, 3)
    check(attend(rows=0, q=None, out=None, positions=None), None)


def select(ctx=REF, logits=P, stride=100, scores=P, groups=2, beams=4, vocabulary=100, best=8, out=P, parents=P, tokens=2 * P):
    return call("rlq_beam_select", ctx, logits, stride, scores, groups, beams, vocabulary, best, out, parents, tokens, None)


def test_select():
    check(select(ctx=None), "InvalidArgument")
    for k in ("logits", "scores", "out", "parents", "tokens"):
        check(select(**{k: None}), "InvalidArgument")
        check(select(**{k: P + 2}), "InvalidArgument")
    check(select(tokens=P), "InvalidArgument")
    check(select(beams=0), "InvalidMatrixShape", 0, 100)
    check(select(vocabulary=0), "InvalidMatrixShape", 4, 0)
    check(select(beams=65), "Unimplemented", 65, 64)
    check(select(vocabulary=2 ** 31), "Unimplemented", 2 ** 31, 2 ** 31 - 1)
    check(select(best=0), "Shape", 0, 400)
    check(select(vocabulary=3, best=13), "Shape", 13, 12)
    check(select(best=65), "Unimplemented", 65, 64)
    check(select(groups=65536), "Unimplemented", 65536, 65535)
    check(select(stride=99), "InvalidLength", 100, 99)
    check(select(groups=0, logits=None), None)


def test_reorder():
    check(reorder(ctx=None), "InvalidArgument")
    check(reorder(null_cache=True), "InvalidArgument")
    check(reorder(n=0), "InvalidArgument")
    for k in ("parents", "lengths", "tables"):
        check(reorder(**{k: None}), "InvalidArgument")
        check(reorder(**{k: P + 2}), "InvalidArgument")
    check(reorder(beams=0), "InvalidMatrixShape", 2, 0)
    check(reorder(beams=33), "Unimplemented", 33, 32)
    check(reorder(groups=65536), "Unimplemented", 65536, 65535)
    check(reorder(width=2 ** 31), "Unimplemented", 2 ** 31, 2 ** 31 - 1)
    e = reorder(caches=[cache(), cache(dtype=BF16)])
    assert (e.code, e.dtype) == (NAMES["Unsupported"], BF16)
    for other in (cache(kv_heads=1), cache(pages=6), cache(k_stride=8192), cache(v_stride=8192), cache(dim=32),
                  cache(page=32, k_stride=8192, v_stride=8192)):
        check(reorder(caches=[cache(), cache(), other]), "Shape", 2, 3)
    check(reorder(groups=0, parents=None), None)
