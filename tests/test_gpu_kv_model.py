"""Several requests of a Llama model decoded together over paged caches, with the framework's
norms and products between the paged calls, against rlq_llama_step on each request alone."""
import numpy as np
import pytest

from llama_fixture import make_config, make_tensors
from rlq_loader import load
from test_gpu_kv import cuda, say
from test_gpu_llama import gpu_config

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch
DT = rlq.DType


class Paged:
    """The model's layers over one paged cache a layer."""

    def __init__(self, ctx, cfg, t, dtype, requests, page, width):
        self.ctx, self.cfg = ctx, cfg
        W, F, kv = cfg.width, cfg.feed_forward, cfg.kv_width
        mat = lambda data, rows, cols: rlq.Weights(ctx, DT(cfg.weight_type), data, rows, cols)  # noqa: E731
        self.layers = [{"n1": cuda(L["attention_norm"]), "n2": cuda(L["feed_forward_norm"]),
                        "qkv": mat(np.concatenate([L["query"], L["key"], L["value"]]), W + 2 * kv, W),
                        "o": mat(L["attention_output"], W, W), "gate": mat(L["gate"], F, W), "up": mat(L["up"], F, W),
                        "down": mat(L["down"], W, F),
                        "cache": rlq.KvCache.make(dtype, requests * width, cfg.kv_heads, page, cfg.head_dim)} for L in t["layers"]]
        self.norm, self.head = cuda(t["output_norm"]), rlq.Weights(ctx, DT(cfg.output_type), t["output"], cfg.vocabulary, W)
        half = cfg.head_dim // 2
        self.freqs = cuda((float(cfg.rope_base) ** (-np.arange(half) / half)).astype(np.float32))
        self.page = page
        i32 = dict(dtype=torch.int32, device="cuda")
        self.tables, self.free = torch.full((requests, width), -1, **i32), torch.arange(requests * width, **i32)
        self.lengths, self.count = torch.zeros(requests, **i32), torch.full((1,), requests * width, **i32)

    def step(self, hidden, new):
        """hidden [rows, width] of the requests' new tokens, in order -> logits [rows, vocabulary]."""
        ctx, c, eps = self.ctx, self.cfg, float(self.cfg.rms_epsilon)
        n, H, K, D = hidden.shape[0], c.heads, c.kv_heads, c.head_dim
        self.lengths, self.count, _, slots, positions, requests = ctx.kv_pages(
            self.lengths, new, self.tables, self.free, self.count, self.page, n)
        one, ids = torch.ones((n, 1), device="cuda"), torch.zeros((n, 1), dtype=torch.int32, device="cuda")
        for L in self.layers:
            _, y, _ = ctx.rms_norm(hidden, L["n1"], eps)
            x = ctx.matmul(L["qkv"], y).view(n, H + 2 * K, D)
            q = ctx.kv_store(L["cache"], x[:, H:H + K], x[:, H + K:], slots, x[:, :H], positions, self.freqs, out=x[:, :H])
            a = ctx.kv_attention(L["cache"], q, self.tables, positions, requests)
            hidden, y, _ = ctx.rms_norm(ctx.matmul(L["o"], a.view(n, H * D)), L["n2"], eps, residual=hidden)
            hidden = ctx.moe_ffn(L["gate"], L["up"], L["down"], y, ids, one, residual=hidden)
        return ctx.matmul(self.head, ctx.rms_norm(hidden, self.norm, eps)[1])


# A token's logits in the two ways differ by the order of f32 sums (some 1e-7), and where such a difference moves a value over
# the border between two of its 8-bit levels by a level: 1/127 of the block's largest value, about 1/40 of a
# vector of 256 values' root mean square, in one value: 1/40 / 16 of the vector's norm.  Two layers have six such
# vectors a token, and a flip in each of them would be sqrt(6) / 640 = 4e-3.
NORM = 4e-3


@pytest.mark.parametrize("dtype,more", [(DT.F32, 0.0), (DT.F16, 2.0 ** -10), (DT.BF16, 2.0 ** -7), (DT.Q8_0, 2.0 ** -6)])
def test_requests_decoded_together(dtype, more):
    """f32 pages hold what the model's own cache holds; the others round keys and values by at most `more` / 2 of their size (of
    a block's largest), which the layers carry to the logits in about that size."""
    say("requests together", dtype)
    ctx = rlq.Context(0)
    cfg = make_config(max_context=64)
    t = make_tensors(cfg, 11)
    model = rlq.LlamaModel(ctx, gpu_config(cfg), t)
    rng = np.random.default_rng(12)
    n, steps = 3, 30
    prompts = [20, 1, 7]  # request r's tokens before the steps
    tokens = [rng.integers(0, cfg.vocabulary, p + steps) for p in prompts]
    want, hidden = [], []
    for r in range(n):
        model.truncate(0)
        logits, rows = [], []
        for pos, token in enumerate(tokens[r]):
            h = model.embedding(int(token))
            rows.append(h.clone())
            logits.append(model.step(h, pos, embedding=False)[1].clone())
        ctx.sync()
        want.append(torch.stack(logits))
        hidden.append(torch.stack(rows))
    paged = Paged(ctx, cfg, t, dtype, n, 16, 4)

    def check(got, r, pos):
        w = want[r][pos]
        assert float((got - w).norm() / w.norm()) <= NORM + more, (r, pos)

    got = paged.step(torch.cat([hidden[r][:prompts[r]] for r in range(n)]), cuda(np.array(prompts, np.int32)))
    ctx.sync()
    at = 0
    for r in range(n):
        for pos in range(prompts[r]):
            check(got[at + pos], r, pos)
        at += prompts[r]
    for k in range(steps):
        got = paged.step(torch.stack([hidden[r][prompts[r] + k] for r in range(n)]), torch.ones(n, dtype=torch.int32, device="cuda"))
        ctx.sync()
        for r in range(n):
            check(got[r], r, prompts[r] + k)
    model.close()
    ctx.close()
