"""Refusals of the norm, router and expert entry points (rlq_rms_norm,
rlq_moe_route, rlq_moe_ffn), which come before any device work: no GPU is needed.
The handles are stand-ins holding the fields that the checks read; no pointer is
followed on these paths."""
import ctypes

import pytest

from rlq_loader import load

rlq = load()
NAMES = {v: k for k, v in rlq.ERROR_NAMES.items()}
P = 4096  # an aligned address that nothing reads
Q8_0, Q4_K, Q5_K, Q6_K, Q8_K = 8, 12, 13, 14, 15


class FakeContext(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("rest", ctypes.c_uint8 * 1024)]


class FakeWeights(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint64),
                ("cols", ctypes.c_uint64), ("dev", ctypes.c_void_p), ("bytes", ctypes.c_uint64),
                ("n2", ctypes.c_uint64), ("n3", ctypes.c_uint64), ("mat_bytes", ctypes.c_uint64)]


CTX = FakeContext()


def call(name, *args):
    err = rlq._Err()
    rc = getattr(rlq.lib(), name)(*args, ctypes.byref(err))
    assert rc == err.code
    return err


def check(err, name, a=0, b=0):
    assert (err.code, err.a, err.b) == (NAMES[name] if name else 0, a, b)


def norm(ctx=ctypes.byref(CTX), x=P, residual=None, weight=P, rows=4, cols=512, eps=1e-5, total=None, y=P, q_dtype=0,
         q=None):
    return call("rlq_rms_norm", ctx, x, residual, weight, rows, cols, eps, total, y, q_dtype, q, None)


def test_rms_norm():
    check(norm(ctx=None), "InvalidArgument")
    check(norm(x=None), "InvalidArgument")
    check(norm(weight=None), "InvalidArgument")
    check(norm(y=None), "InvalidArgument")  # nothing to write
    check(norm(total=P, y=P), "InvalidArgument")
    check(norm(x=P + 2), "InvalidArgument")
    check(norm(residual=P + 1), "InvalidArgument")
    check(norm(q=P + 2, q_dtype=Q8_K), "InvalidArgument")
    check(norm(q=P + 1, q_dtype=Q8_0), "InvalidArgument")
    check(norm(q=P, q_dtype=99), "InvalidType")
    check(norm(q=P, q_dtype=Q4_K), "Unimplemented")
    check(norm(q=P, q_dtype=Q8_K, cols=300), "NonMultiple", 300, 256)
    check(norm(q=P, q_dtype=Q8_0, cols=48), "NonMultiple", 48, 32)
    check(norm(cols=0), "InvalidMatrixShape", 4, 0)
    for eps in (0.0, -1e-5, float("inf"), float("nan")):
        check(norm(eps=eps), "InvalidConfig", 2)
    check(norm(cols=32769), "Unimplemented", 32769, 32768)
    check(norm(rows=65536), "Unimplemented", 65536, 65535)
    check(norm(rows=0, x=None, weight=None, y=None), None)  # an empty call


def route(ctx=ctypes.byref(CTX), router=P, x=P, tokens=3, cols=64, experts=8, slots=2, flags=0, scale=1.0, bias=None,
          ids=P, weights=P, logits=None):
    return call("rlq_moe_route", ctx, router, x, tokens, cols, experts, slots, flags, scale, bias, ids, weights, logits,
                None)


def test_moe_route():
    check(route(ctx=None), "InvalidArgument")
    for k in ("router", "x", "ids", "weights"):
        check(route(**{k: None}), "InvalidArgument")
        check(route(**{k: P + 2}), "InvalidArgument")
    check(route(bias=P + 2), "InvalidArgument")
    check(route(logits=P + 2), "InvalidArgument")
    check(route(flags=4), "InvalidArgument", 4)
    check(route(cols=0), "InvalidMatrixShape", 8, 0)
    check(route(experts=0), "InvalidMatrixShape", 0, 64)
    check(route(slots=0), "Shape", 0, 8)
    check(route(slots=9), "Shape", 9, 8)
    check(route(experts=1025), "Unimplemented", 1025, 1024)
    check(route(experts=100, slots=65), "Unimplemented", 65, 64)
    check(route(tokens=65536), "Unimplemented", 65536, 65535)
    check(route(cols=2 ** 30 + 4), "Unimplemented", 2 ** 30 + 4, 2 ** 30)
    check(route(tokens=0, ids=None), None)


def matrix(dtype=Q4_K, rows=512, cols=256, n2=4, n3=1, device=0):
    return FakeWeights(device, dtype, rows, cols, P, 0, n2, n3, 0)


def ffn(ctx=ctypes.byref(CTX), gate=None, up=None, down=None, x_dtype=0, x=P, tokens=2, ids=P, weights=P, slots=2,
        residual=None, y=P):
    gate, up = gate or matrix(), up or matrix()
    down = down or matrix(rows=256, cols=512)
    refs = [None if m == "null" else ctypes.byref(m) for m in (gate, up, down)]
    return call("rlq_moe_ffn", ctx, *refs, x_dtype, x, tokens, ids, weights, slots, residual, y, None)


def test_moe_ffn():
    check(ffn(ctx=None), "InvalidArgument")
    for k in ("gate", "up", "down"):
        check(ffn(**{k: "null"}), "InvalidArgument")
    check(ffn(up=matrix(device=1)), "InvalidArgument")
    check(ffn(gate=matrix(n3=2)), "Shape", 4, 4)
    check(ffn(up=matrix(n2=5)), "Shape", 4, 5)
    check(ffn(down=matrix(rows=256, cols=512, n2=3)), "Shape", 4, 3)
    check(ffn(up=matrix(rows=544)), "Shape", 544, 256)
    check(ffn(up=matrix(cols=512)), "Shape", 512, 512)
    check(ffn(down=matrix(rows=256, cols=768)), "Shape", 256, 768)
    check(ffn(slots=0), "Shape", 0, 4)
    e = ffn(up=matrix(dtype=Q6_K))
    assert (e.code, e.dtype) == (NAMES["Unsupported"], Q6_K)
    e = ffn(x_dtype=Q8_0)
    assert (e.code, e.dtype) == (NAMES["Unsupported"], Q8_0)
    check(ffn(gate=matrix(n2=1025), up=matrix(n2=1025), down=matrix(rows=256, cols=512, n2=1025)), "Unimplemented", 1025,
          1024)
    check(ffn(slots=65), "Unimplemented", 65, 64)
    check(ffn(tokens=65536), "Unimplemented", 65536, 65535)
    for k in ("x", "ids", "weights", "y"):
        check(ffn(**{k: None}), "InvalidArgument")
        check(ffn(**{k: P + 2}), "InvalidArgument")
    check(ffn(residual=P + 1), "InvalidArgument")
    check(ffn(x=P + 8), "InvalidArgument")
    check(ffn(x=P + 2, x_dtype=Q8_K), "InvalidArgument")
    check(ffn(tokens=0, x=None, y=None), None)
    # a grid that would not fit
    wide = dict(gate=matrix(rows=2 ** 30, n2=64), up=matrix(rows=2 ** 30, n2=64),
                down=matrix(rows=256, cols=2 ** 30, n2=64))
    check(ffn(tokens=32, **wide), "Unimplemented", 2 ** 30, 256)


@pytest.mark.parametrize("name,args", [("rlq_rms_norm", (None, None, None, None, 0, 0, 0.0, None, None, 0, None, None)),
                                       ("rlq_moe_route", (None, None, None, 0, 0, 0, 0, 0, 0.0, None, None, None, None, None)),
                                       ("rlq_moe_ffn", (None, None, None, None, 0, None, 0, None, None, 0, None, None, None))])
def test_no_error_record_is_needed(name, args):
    assert getattr(rlq.lib(), name)(*args, None) == NAMES["InvalidArgument"]
