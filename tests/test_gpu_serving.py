"""Decoder layers over the paged cache as a server runs them: quantized projections with the requests' adapters, append,
attention and the output projection, over prompts, forks, captured decode steps, rejected tokens and compaction.

Every stage is checked against the 64-bit formula on the stage's own inputs, with the tolerances of the single
operators' tests; what a layer hands on is what the next one gets.
"""
import math

import numpy as np
import pytest

from test_gpu_adapters import _check, _load
from test_gpu_batch import U, Model, env  # noqa: F401  (env: the fixture)

pytestmark = pytest.mark.gpu

LAYERS, KV, GROUP, DIM, HIDDEN = 2, 2, 3, 64, 224
QW, KW = KV * GROUP * DIM, KV * DIM


class Decoder:
    def __init__(self, env, kind, fmt):
        self.sat, self.torch, self.ctx = sat, torch, ctx = env
        self.m = Model(env, kind, DIM, KV, GROUP, 16, pages=96, layers=LAYERS, rope=1e4, seed=5)
        self.rows = sat.AdapterRows(ctx)
        self.layers = []
        for i in range(LAYERS):
            qkv = self.projection(QW + 2 * KW, HIDDEN, fmt, 2 * i)
            self.layers.append((qkv, self.projection(HIDDEN, QW, fmt, 2 * i + 1)))

    def projection(self, rows, cols, fmt, seed):
        """(quantized matrix, its adapters, their weights, the payload to keep)"""
        from satori_b200 import _lib
        sat, torch, f = self.sat, self.torch, getattr(self.sat, fmt)
        w = self.m.normal(rows * cols) * 0.06
        payload = torch.empty(rows * (cols // 32) * (34 if f == sat.Q8_0 else 18), dtype=torch.uint8, device="cuda")
        _lib.check(_lib.lib().satori_quantize_q_device(self.ctx.handle, w.data_ptr(), rows, cols, f, payload.data_ptr()))
        matrix = sat.CudaQuantizedMatrix.from_device(self.ctx, payload.data_ptr(), payload.numel(), rows, cols, f)
        adapters = sat.AdapterSet(rows, cols, 3, 16, dtype="bf16", ctx=self.ctx)
        return matrix, adapters, _load(torch, adapters, "bf16", rows, cols, [16, 4, 9], seed), payload

    def buffers(self, n):
        torch = self.torch
        f32 = lambda w: torch.full((n, w), math.nan, device="cuda")
        return [dict(x=f32(HIDDEN), qkv=f32(QW + 2 * KW), q=torch.empty((n, QW), dtype=self.m.dtype, device="cuda"),
                     att=f32(QW), o=f32(HIDDEN)) for _ in range(LAYERS + 1)]

    def run(self, bufs):
        for layer, ((wqkv, aqkv, _, _), (wo, ao, _, _)) in enumerate(self.layers):
            b = bufs[layer]
            aqkv.execute_device(wqkv, self.rows, b["x"], b["qkv"])
            q, k, v = b["qkv"].split([QW, KW, KW], 1)
            self.m.batch.append_device(layer, k, v, q, b["q"])
            self.m.batch.attention_device(layer, b["q"], b["att"])
            ao.execute_device(wo, self.rows, b["att"], b["o"])
            self.torch.add(b["x"], b["o"], out=bufs[layer + 1]["x"])

    def check(self, bufs, seqs, counts, ids):
        torch, m = self.torch, self.m
        n = sum(counts)
        starts = [m.cache.length(s) - c for s, c in zip(seqs, counts)]
        positions = np.concatenate([np.arange(a, a + c) for a, c in zip(starts, counts)])
        eps = torch.finfo(m.dtype).eps / 2
        tiny = torch.finfo(m.dtype).smallest_normal * eps * 2
        for s in seqs:
            m.tokens[s] = m.read(s)
        from satori_b200 import _lib
        for layer, ((wqkv, _, lqkv, _), (wo, _, lo, _)) in enumerate(self.layers):
            b = bufs[layer]
            for matrix, x, out, weights in ((wqkv, b["x"], b["qkv"], lqkv), (wo, b["att"], b["o"], lo)):
                base = torch.empty_like(out)
                matrix.execute_device(x.data_ptr(), base.data_ptr(), n, _lib.ORDER_BATCH)
                _check(torch, out, x, base, ids, weights)
            assert torch.equal(bufs[layer + 1]["x"], b["x"] + b["o"])
            qkv = b["qkv"].double().cpu().numpy().reshape(n, -1, DIM)
            exact = m.rotate(qkv[:, :KV * (GROUP + 1)], positions)
            slack = 2.0 ** -40 * np.abs(qkv).max() + tiny
            q = b["q"].double().cpu().numpy().reshape(n, KV * GROUP, DIM)
            assert np.all(np.abs(q - exact[:, :KV * GROUP]) <= eps * np.abs(exact[:, :KV * GROUP]) + slack)
            got = b["att"].double().cpu().numpy().reshape(n, KV, GROUP, DIM)
            row = 0
            for s, a, c in zip(seqs, starts, counts):
                k, v = m.tokens[s][:, layer]
                for held, new in ((k, exact[row:row + c, KV * GROUP:]), (v, qkv[row:row + c, KV * (GROUP + 1):])):
                    assert np.all(np.abs(held[a:a + c] - new) <= eps * np.abs(new) + slack)
                for r in range(c):
                    t = a + r + 1
                    out, size, scores = m.formula(q[row].reshape(KV, GROUP, DIM), k[:t], v[:t])
                    tol = (2 * (DIM + 4) * scores[..., None] + 2 * (t + 16)) * U * size
                    if m.kind != "f32":
                        tol = tol + eps * size
                    assert np.all(np.abs(got[row] - out) <= tol), (layer, s, r)
                    row += 1

    def step(self, seqs, counts, adapters):
        ids = np.repeat(adapters, counts)
        self.m.batch.step(seqs, counts)
        self.rows.assign(ids)
        bufs = self.buffers(sum(counts))
        bufs[0]["x"].copy_(self.m.normal(sum(counts), HIDDEN))
        self.run(bufs)
        self.check(bufs, seqs, counts, ids)


@pytest.mark.parametrize("kind,fmt", [("f32", "Q8_0"), ("bf16", "Q4_0"), ("f16", "Q8_0")])
def test_layers_of_a_server(env, kind, fmt):  # noqa: F811
    sat, torch, ctx = env
    d = Decoder(env, kind, fmt)
    m = d.m
    root = m.new()
    d.step([root], [300], [-1])                                # an instruction that the requests share
    a, b, c = m.fork([root] * 3, [300, 288, 41])               # whole pages shared, a page copied, a page cut
    d.step([a, b, c], [1, 20, 75], [0, 1, -1])                 # one decodes, two bring their prompts
    seqs, ids = [c, a, b], np.array([2, 0, 1])

    # Decode steps: captured once, planned and assigned outside.
    bufs = d.buffers(3)
    m.batch.step(seqs, [1] * 3)
    d.rows.assign(ids)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            d.run(bufs)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    for step in range(4):
        if step:
            ids = np.roll(ids, 1) if step == 2 else ids
            m.batch.step(seqs, [1] * 3)
            d.rows.assign(ids)
        bufs[0]["x"].copy_(m.normal(3, HIDDEN))
        graph.replay()
        torch.cuda.synchronize()
        d.check(bufs, seqs, [1] * 3, ids)

    # Four drafted tokens each; one request keeps two of them, one ends, the others' pages move together.
    d.step(seqs, [4] * 3, ids)
    m.cache.rewind([a], [m.cache.length(a) - 2])
    m.cache.free([b, root])
    kept = {s: m.read(s) for s in (a, c)}
    free = m.cache.info()["free"]
    m.cache.compact()
    assert m.cache.info()["free"] == free
    for s, was in kept.items():
        assert np.array_equal(m.read(s), was)
    d.step([a, c], [1, 3], [0, 1])
