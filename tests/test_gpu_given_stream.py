"""Calls on a stream that is given, while torch's current one is busy: tensors that
a call makes itself (its outputs, the copy of a strided x) must not be memory that the
current stream still uses, nor be filled by it."""
import numpy as np
import pytest

from llama_fixture import make_config, make_tensors
from rlq_loader import load
from test_gpu_llama import gpu_config
from test_gpu_sweep import _weights

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType


def normal(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32)).cuda()


def stack(ctx, rows, cols, n=4):
    return rlq.Weights(ctx, DT.Q6_K, _weights(DT.Q6_K, n * rows, cols, 3), rows, cols, n)


def calls(ctx):
    """name -> call(stream), a tuple of outputs"""
    W, one, down = stack(ctx, 256, 256), stack(ctx, 256, 256, 1), stack(ctx, 256, 256)
    x, w = normal(1, 3, 256), normal(2, 256)
    ids = torch.tensor([[0, 1], [2, 3], [1, 1]], dtype=torch.int32, device="cuda")
    weights, router = normal(3, 3, 2), normal(4, 8, 256)
    strided = normal(5, 3, 2, 256).transpose(0, 1)
    cfg = make_config(n_layers=1, vocabulary=500, max_context=8)
    model = rlq.LlamaModel(ctx, gpu_config(cfg), make_tensors(cfg, 7))

    def llama(s):
        model.truncate(0)
        h = model.embedding(5, stream=s)
        return (h,) + model.step(h, 0, argmax=True, stream=s) + model.intermediates(stream=s)

    return {
        "llama": llama,
        "rms_norm": lambda s: ctx.rms_norm(x, w, 1e-5, residual=x, packed=DT.Q8_K, stream=s),
        "moe_route": lambda s: ctx.moe_route(router, x, 2, logits=True, stream=s),
        "moe_route strided": lambda s: ctx.moe_route(router, strided, 2, logits=True, stream=s),
        "moe_ffn": lambda s: (ctx.moe_ffn(W, W, down, x, ids, weights, stream=s),),
        "matmul": lambda s: (ctx.matmul(one, x, stream=s),),
        "matmul strided": lambda s: (ctx.matmul(one, strided, stream=s),),
        "multiply": lambda s: (ctx.multiply(one, x[0], stream=s),),
        "matmul_argmax": lambda s: ctx.matmul_argmax(one, x, stream=s),
        "quantize": lambda s: (ctx.quantize(DT.Q8_K, x, stream=s),),
        "quantize strided": lambda s: (ctx.quantize(DT.Q8_K, strided, stream=s),),
        "mul_mat": lambda s: (ctx.mul_mat(one, x.view(1, 1, 3, 256), stream=s),),
        "mul_mat_id": lambda s: (ctx.mul_mat_id(W, x.view(3, 1, 256), ids, stream=s),),
        "block_sums": lambda s: ctx.block_sums(one, x, stream=s),
        "block_sums_ex": lambda s: ctx.block_sums_ex(one, x, stream=s),
    }


@pytest.mark.parametrize("handle", [False, True], ids=["stream", "handle"])
@pytest.mark.parametrize("name", ["rms_norm", "moe_route", "moe_route strided", "moe_ffn", "matmul", "matmul strided", "multiply",
                                  "matmul_argmax", "quantize", "quantize strided", "mul_mat", "mul_mat_id", "block_sums",
                                  "block_sums_ex", "llama"])
def test_tensors_of_a_call_on_a_given_stream(name, handle):
    print("[case] given stream", name, handle, flush=True)
    ctx = rlq.Context(0)
    call = calls(ctx)[name]
    want = call(None)
    ctx.sync()
    s = torch.cuda.Stream()
    at = s.cuda_stream if handle else s
    call(at)  # the scratch is there
    big = torch.ones((8192, 8192), device="cuda")
    out = torch.mm(big, big)
    torch.cuda.synchronize()
    # free memory of these sizes, in use by the current stream until its queue is done
    sizes = [k * 512 for k in (1, 2, 4, 6, 8, 12, 16, 24)] + [t.numel() * t.element_size() for t in want]
    taken = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(64)]
    torch.cuda.synchronize()
    for _ in range(20):  # (20 products of 1.1e12 operations)
        torch.mm(big, big, out=out)
    for k in range(len(taken)):
        taken[k].fill_(7)
    taken = taken[::2]  # (every other, so that what is free stays in pieces of these sizes)
    got = call(at)
    s.synchronize()
    busy = not torch.cuda.current_stream().query()
    torch.cuda.synchronize()
    assert busy  # (the call did not wait for the current stream)
    ctx.sync()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ctx.sync()
    for a, b in zip(call(0), want):  # HIP's null stream
        assert torch.equal(a, b)
    ctx.sync()
    ctx.close()
