"""A decode batch over a paged cache on the GPU: append, page copies and attention against 64-bit formulas.

Tolerances, derived from the operations (u = 2^-24, the unit roundoff of FP32):

* append rotates in FP64 and rounds once: half a step of the output's type, plus 2^-40 of the magnitude for the
  differences of two FP64 sin / cos implementations.
* attention, in FP32: a score is a sum of d products, in error by at most (d + 4) u S, S = sum |q k| / sqrt(d)
  (the products, their sum, the scaling); it moves a weight by that much relative to it, in the numerator and
  in the denominator, and the exponential and the sums over the T keys add (T + 16) u each:
  |err| <= (2 (d + 4) S + 2 (T + 16)) u W, W = sum_t p_t |v_t|.
  In a 16-bit cache the weights may be rounded to its type before they meet v: half a step (eps / 2) of W, and
  the result to its own type: half a step of it.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def env():
    from satori_b200 import build
    build.build()
    import torch

    import satori_b200 as sat
    ctx = sat.Context(0)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    yield sat, torch, ctx
    ctx.close()


def _dtype(torch, kind):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


class Model:
    """A paged cache with the tokens of every sequence kept beside it (float64), unwritten memory NaN."""

    def __init__(self, env, kind, dim, kv_heads, group, page, pages=64, layers=2, rope=0.0, rotary=0, seed=0):
        self.sat, self.torch, self.ctx = env
        torch = self.torch
        self.kind, self.dim, self.kv, self.group, self.page, self.layers = kind, dim, kv_heads, group, page, layers
        self.dtype = _dtype(torch, kind)
        self.pool = torch.full((layers, pages, 2, kv_heads, page, dim), math.nan, dtype=self.dtype, device="cuda")
        self.cache = self.sat.PagedCache(layers, pages, page, kv_heads, dim, dtype=kind, memory=self.pool, ctx=self.ctx)
        self.batch = self.sat.DecodeBatch(self.cache, kv_heads * group, rope, rotary)
        self.rope, self.rotary = rope, (rotary or dim) if rope else 0
        self.rng = np.random.default_rng(seed)
        self.tokens = {}                                      # id -> [2, layers, tokens, kv, dim] float64

    def normal(self, *shape):
        return self.torch.from_numpy(self.rng.standard_normal(shape, dtype=np.float32)).cuda()

    def new(self):
        s = self.cache.create(1)[0]
        self.tokens[s] = np.zeros((2, self.layers, 0, self.kv, self.dim))
        return s

    def fork(self, parents, positions, share=True):
        ids = (self.cache.fork if share else self.cache.copy)(parents, positions)
        for c, p, n in zip(ids, parents, positions):
            self.tokens[c] = self.tokens[p][:, :, :n].copy()
        return ids

    def rotate(self, x, positions):
        """RopeHalf in float64 on [rows, heads, dim]."""
        if not self.rotary:
            return x
        half = self.rotary // 2
        angle = positions[:, None] / self.rope ** (2.0 * np.arange(half) / self.rotary)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        out = x.copy()
        a, b = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, a * s + b * c
        return out

    def step(self, seqs, counts, q_scale=1.0, in_type=None, check_append=True):
        """Steps, appends in every layer, and returns the rotated queries of each layer (device)."""
        torch = self.torch
        self.batch.step(seqs, counts)
        n, qh = sum(counts), self.kv * self.group
        starts = [self.tokens[s].shape[2] for s in seqs]
        positions = np.concatenate([np.arange(a, a + c) for a, c in zip(starts, counts)]) if n else np.zeros(0)
        queries, written = [], []
        for layer in range(self.layers):
            qkv = self.normal(n, (qh + 2 * self.kv) * self.dim) * q_scale
            qkv = qkv.to(in_type or torch.float32)
            q, k, v = qkv.split([qh * self.dim, self.kv * self.dim, self.kv * self.dim], 1)
            q_out = torch.empty((n, qh * self.dim), dtype=self.dtype, device="cuda")
            self.batch.append_device(layer, k, v, q, q_out)
            x = qkv.double().cpu().numpy().reshape(n, qh + 2 * self.kv, self.dim)
            exact = self.rotate(x[:, :qh + self.kv], positions)
            eps = torch.finfo(self.dtype).eps / 2
            tiny = torch.finfo(self.dtype).smallest_normal * eps * 2      # half a subnormal step and more
            slack = 2.0 ** -40 * np.abs(x[:, :qh + self.kv]).max(initial=1.0)
            got = q_out.double().cpu().numpy().reshape(n, qh, self.dim)
            if check_append:
                assert np.all(np.abs(got - exact[:, :qh]) <= eps * np.abs(exact[:, :qh]) + slack + tiny)
            queries.append(q_out)
            written.append((exact[:, qh:], x[:, qh + self.kv:], slack + tiny, eps))
        row = 0
        for s, a, c in zip(seqs, starts, counts):
            stored = self.read(s)                             # what the cache holds is what attention reads
            for layer, (k, v, slack, eps) in enumerate(written):
                for j, x in enumerate((k, v)):
                    new = stored[j, layer, a:a + c]
                    exact = x[row:row + c]
                    if check_append:
                        assert np.all(np.abs(new - exact) <= eps * np.abs(exact) + slack)
            assert np.array_equal(stored[:, :, :a], self.tokens[s])       # earlier tokens are untouched
            self.tokens[s] = stored
            row += c
        return queries

    def read(self, s):
        n = self.cache.length(s)
        table = self.torch.from_numpy(self.cache.table(s).astype(np.int64)).cuda()
        held = self.pool[:, table].double()                   # [layer, page, 2, kv, token, dim]
        held = held.permute(2, 0, 1, 4, 3, 5).reshape(2, self.layers, -1, self.kv, self.dim)
        return held[:, :, :n].cpu().numpy()

    def check(self, seqs, counts, queries, out_f32=False, strided=False):
        torch = self.torch
        qh, n = self.kv * self.group, sum(counts)
        for layer, q in enumerate(queries):
            kind = torch.float32 if out_f32 else self.dtype
            if strided:                                       # odd row strides: no wide accesses
                big_q = torch.zeros((n, qh * self.dim + 3), dtype=self.dtype, device="cuda")
                big_q[:, 3:] = q
                big = torch.full((n, qh * self.dim + 5), 7.0, dtype=kind, device="cuda")
                q_in, out = big_q[:, 3:], big[:, 1:1 + qh * self.dim]
            else:
                q_in, out = q, torch.full((n, qh * self.dim), math.nan, dtype=kind, device="cuda")
            self.batch.attention_device(layer, q_in, out)
            got = out.double().cpu().numpy().reshape(n, self.kv, self.group, self.dim)
            if strided:
                assert bool((big[:, 0] == 7).all()) and bool((big[:, 1 + qh * self.dim:] == 7).all())
            qd = q.double().cpu().numpy().reshape(n, self.kv, self.group, self.dim)
            row = 0
            for s, c in zip(seqs, counts):
                k, v = self.tokens[s][:, layer]
                for r in range(c):
                    t = k.shape[0] - c + r + 1
                    exact, size, scores = self.formula(qd[row], k[:t], v[:t])
                    tol = (2 * (self.dim + 4) * scores[..., None] + 2 * (t + 16)) * U * size
                    if self.kind != "f32":
                        half = torch.finfo(self.dtype).eps / 2
                        tol = tol + half * size + (0 if out_f32 else half * np.abs(exact) +
                                                   torch.finfo(self.dtype).smallest_normal * half * 2)
                    err = np.abs(got[row] - exact)
                    assert np.all(err <= tol), (s, r, t, float(np.nanmax(err / tol)), bool(np.isnan(got[row]).any()))
                    row += 1

    @staticmethod
    def formula(q, k, v):
        """(out, sum p |v|, max_t sum |q k| / sqrt(d)) for one row: q [kv, group, dim], k and v [t, kv, dim]."""
        scale = 1 / math.sqrt(q.shape[-1])
        s = np.einsum("hgd,thd->hgt", q, k) * scale
        size = (np.einsum("hgd,thd->hgt", np.abs(q), np.abs(k)) * scale).max(-1)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        return np.einsum("hgt,thd->hgd", p, v), np.einsum("hgt,thd->hgd", p, np.abs(v)), size


KINDS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300])
def test_single_sequence_lengths(env, kind, length):
    m = Model(env, kind, 64, 2, 3, 16)
    s = m.new()
    if length > 1:
        m.step([s], [length - 1])
    q = m.step([s], [1])
    m.check([s], [1], q)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 4, 7), (128, 2, 6), (64, 8, 1), (96, 2, 5), (256, 1, 8),
                                                (8, 3, 2), (72, 1, 9), (128, 1, 40)])
def test_head_layouts(env, kind, dim, kv_heads, group):
    """Ragged sequences, some without new rows in the step, a prompt chunk beside single tokens."""
    m = Model(env, kind, dim, kv_heads, group, 32, layers=1, seed=dim + group)
    seqs = [m.new() for _ in range(5)]
    m.step(seqs, [40, 0, 129, 7, 90])
    counts = [1, 3, 1, 0, 70]
    q = m.step(seqs, counts)
    m.check(seqs, counts, q)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_shared_prefix_and_nested_forks(env, kind, page, dim):
    """A prompt shared by all, a branch shared by some, tails of their own; forks inside a page."""
    m = Model(env, kind, dim, 2, 6, page, pages=max(48, 4096 // page), layers=1, seed=page)
    root = m.new()
    m.step([root], [777])
    a, b, c = m.fork([root] * 3, [777, 768, 700])
    m.step([a], [300])
    d, e = m.fork([a, a], [1077, 1024])
    seqs = [e, b, a, c, d]
    m.step([b, d], [5, 17])
    counts = [1, 1, 2, 33, 1]
    q = m.step(seqs, counts)
    assert m.batch.info()["segments"] >= 7
    m.check(seqs, counts, q)


@pytest.mark.parametrize("kind", KINDS)
def test_many_rows_behind_a_prefix(env, kind):
    """More rows than a tile holds, in the shared part and in the prompts."""
    m = Model(env, kind, 128, 1, 7, 64, pages=80, layers=1, seed=3)
    root = m.new()
    m.step([root], [640])
    seqs = m.fork([root] * 5, [640] * 5)
    counts = [50, 1, 64, 3, 37]
    q = m.step(seqs, counts)
    m.check(seqs, counts, q)


@pytest.mark.parametrize("kind", KINDS)
def test_forked_equals_copied(env, kind):
    """The same tokens through shared and through private pages: both within the tolerance, copies intact."""
    m = Model(env, kind, 128, 2, 4, 16, pages=256, layers=2, seed=4)
    root = m.new()
    m.step([root], [403])
    seqs = m.fork([root] * 2, [403, 390]) + m.fork([root] * 2, [403, 390], share=False)
    q = m.step(seqs, [1] * 4)
    m.check(seqs, [1] * 4, q)


@pytest.mark.parametrize("kind", KINDS)
def test_large_and_tiny_scores(env, kind):
    """Weights concentrated on single keys (scores in the hundreds) and the running maximum rising late."""
    m = Model(env, kind, 64, 1, 4, 16, pages=64, layers=1, seed=9)
    s = m.new()
    m.step([s], [400])
    q = m.step([s], [1], q_scale=20.0)
    m.check([s], [1], q)
    for scale in (1e-3, 30.0, 1.0):
        q = m.step([s], [90], q_scale=scale)
        m.check([s], [90], q)


@pytest.mark.parametrize("kind", KINDS)
def test_strided_rows_and_float_output(env, kind):
    m = Model(env, kind, 64, 2, 2, 16, layers=1, seed=10)
    seqs = [m.new(), m.new()]
    m.step(seqs, [30, 150])
    q = m.step(seqs, [1, 20])
    m.check(seqs, [1, 20], q, strided=True)
    m.check(seqs, [1, 20], q, out_f32=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("same_type", [False, True])
@pytest.mark.parametrize("rotary", [0, 32, 64])
def test_append_rotates_like_ropehalf(env, kind, same_type, rotary):
    sat, torch, ctx = env
    m = Model(env, kind, 64, 3, 2, 16, layers=2, rope=1e4, rotary=rotary, seed=rotary)
    seqs = [m.new(), m.new(), m.new()]
    in_type = _dtype(torch, kind) if same_type else None
    m.step(seqs, [3, 0, 33], in_type=in_type)
    q = m.step(seqs, [40, 1, 1], in_type=in_type)
    m.check(seqs, [40, 1, 1], q)


def test_append_is_bitwise_ropehalf_in_fp32(env):
    """The FP32 cache row equals TransformerOps.rope_half of the key at its position, far positions too."""
    sat, torch, ctx = env
    m = Model(env, "f32", 64, 1, 1, 256, pages=160, layers=1, rope=1e6)
    s = m.new()
    m.cache.extend([s], [40000])
    m.batch.step([s], [2])
    k, v = m.normal(2, 64), m.normal(2, 64)
    m.batch.append_device(0, k, v)
    torch.cuda.synchronize()
    table = m.cache.table(s)
    for r in range(2):
        want = k[r].cpu().numpy().copy()
        sat.TransformerOps.rope_half(want, 64, 40000 + r, 1e6, 64, ctx=ctx)
        at = 40000 + r
        got = m.pool[0, int(table[at // 256]), :, 0, at % 256].cpu().numpy()
        assert np.array_equal(got[0].view(np.uint32), want.view(np.uint32))
        assert np.array_equal(got[1], v[r].cpu().numpy())


def test_append_writes_only_the_new_slots(env):
    sat, torch, ctx = env
    m = Model(env, "bf16", 64, 2, 2, 16, pages=8, layers=2)
    seqs = [m.new(), m.new()]
    m.cache.extend(seqs, [5, 16])
    m.batch.step(seqs, [3, 1])
    before = m.pool.clone()
    m.batch.append_device(1, m.normal(4, 128), m.normal(4, 128))
    changed = ~torch.isnan(m.pool) & torch.isnan(before)
    want = torch.zeros_like(changed)
    for s, a, n in ((seqs[0], 5, 3), (seqs[1], 16, 1)):
        for t in range(a, a + n):
            want[1, int(m.cache.table(s)[t // 16]), :, :, t % 16] = True
    assert torch.equal(changed, want)


def test_values_behind_the_end_and_in_free_pages_never_matter(env):
    """Infinities behind each sequence's end (the pages start as NaN in every other test)."""
    sat, torch, ctx = env
    for kind in KINDS:
        m = Model(env, kind, 128, 1, 4, 64, layers=1)
        m.pool.fill_(math.inf)
        seqs = [m.new(), m.new()]
        m.step(seqs, [3, 65])
        q = m.step(seqs, [1, 2])
        m.check(seqs, [1, 2], q)


@pytest.mark.parametrize("kind", KINDS)
def test_long_cache(env, kind):
    """A cache whose offsets pass 2^31 elements, and keys far into a sequence."""
    sat, torch, ctx = env
    dim, kv, page, pages = 128, 4, 256, 3000
    dtype = _dtype(torch, kind)
    layers = 3                                                # 3 * 3000 * 2 * 4 * 256 * 128 = 2.4e9 elements
    pool = torch.zeros((layers, pages, 2, kv, page, dim), dtype=dtype, device="cuda")
    cache = sat.PagedCache(layers, pages, page, kv, dim, dtype=kind, memory=pool, ctx=ctx)
    batch = sat.DecodeBatch(cache, 4 * kv)
    filler, s = cache.create(2)
    cache.extend([filler], [page * (pages - 80)])             # the sequence's pages come last
    cache.extend([s], [20000 - 1])
    batch.step([s], [1])
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.from_numpy(cache.table(s).astype(np.int64)).cuda()
    assert int(table.min()) == pages - 80
    pool[2, table] = torch.randn((table.numel(), 2, kv, page, dim), generator=g, device="cuda").to(dtype)
    q = torch.randn((1, 4 * kv * dim), generator=g, device="cuda").to(dtype)
    out = torch.empty_like(q)
    batch.attention_device(2, q, out)
    held = pool[2, table].permute(1, 2, 0, 3, 4).reshape(2, kv, -1, dim)[:, :, :20000].double()
    qd = q.double().view(kv, 4, dim)
    score = qd @ held[0].transpose(1, 2) / math.sqrt(dim)
    size = (qd.abs() @ held[0].abs().transpose(1, 2) / math.sqrt(dim)).amax()
    p = torch.softmax(score, -1)
    exact, w = p @ held[1], p @ held[1].abs()
    tol = (2 * (dim + 4) * size + 2 * (20000 + 16)) * U * w
    if kind != "f32":
        half = torch.finfo(dtype).eps / 2
        tol = tol + half * w + half * exact.abs() + torch.finfo(dtype).smallest_normal
    assert bool(((out.double().view(kv, 4, dim) - exact).abs() <= tol).all())


@pytest.mark.parametrize("kind", KINDS)
def test_page_copies_on_the_device(env, kind):
    """Forks, copies, rewinds and compaction move the bytes of every layer; nothing else changes."""
    sat, torch, ctx = env
    m = Model(env, kind, 72, 3, 1, 16, pages=40, layers=3, seed=12)
    a, b = m.new(), m.new()
    m.step([a, b], [100, 33])
    kids = m.fork([a, a, b], [100, 50, 20]) + m.fork([b, a], [33, 7], share=False)
    for s in kids:
        assert np.array_equal(m.read(s), m.tokens[s])
    m.cache.rewind([kids[0], a], [90, 85])                    # inside a shared page
    m.tokens[kids[0]], m.tokens[a] = m.tokens[kids[0]][:, :, :90], m.tokens[a][:, :, :85]
    m.cache.free([b])
    del m.tokens[b]
    before = {s: m.read(s) for s in m.tokens}
    assert m.cache.compact() > 0
    for s, tokens in m.tokens.items():
        assert np.array_equal(before[s], tokens) and np.array_equal(m.read(s), tokens)
    seqs = list(m.tokens)
    q = m.step(seqs, [1] * len(seqs))
    m.check(seqs, [1] * len(seqs), q)


def test_many_page_copies_in_one_call(env):
    """More pairs than one launch takes."""
    sat, torch, ctx = env
    pool = torch.randn((1, 10000, 2, 1, 16, 8), device="cuda")
    cache = sat.PagedCache(1, 10000, 16, 1, 8, memory=pool, ctx=ctx)
    s = cache.create(1)
    cache.extend(s, [16 * 4900 + 3])
    c = cache.copy(s)[0]
    t = [torch.from_numpy(cache.table(x).astype(np.int64)).cuda() for x in (s[0], c)]
    assert t[0].numel() == 4901 and torch.equal(pool[:, t[0]], pool[:, t[1]])


@pytest.mark.parametrize("kind", KINDS)
def test_captured_layers_replay_for_the_next_steps(env, kind):
    """append and attention captured once; each later step is planned outside and the graph replayed."""
    sat, torch, ctx = env
    m = Model(env, kind, 128, 2, 3, 16, pages=64, layers=1, rope=1e4, seed=21)
    root = m.new()
    m.step([root], [270])
    seqs = m.fork([root] * 3, [270, 256, 200])
    m.step(seqs, [1] * 3)
    n, qw, kw = 3, 6 * 128, 2 * 128
    qkv = torch.zeros((n, qw + 2 * kw), device="cuda")
    q, k, v = qkv.split([qw, kw, kw], 1)
    q_out = torch.zeros((n, qw), dtype=m.dtype, device="cuda")
    out = torch.zeros_like(q_out)
    stream = torch.cuda.Stream()
    m.batch.step(seqs, [1] * 3)
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            m.batch.append_device(0, k, v, q, q_out)
            m.batch.attention_device(0, q_out, out)
            with pytest.raises(sat.NotSupportedError):
                m.batch.step(seqs, [1] * 3)
            with pytest.raises(sat.NotSupportedError):
                m.cache.fork([root])
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    at = [x + 1 for x in (270, 256, 200)]
    for step in range(20):
        if step:
            m.batch.step(seqs, [1] * 3)
        qkv.copy_(m.normal(n, qw + 2 * kw))
        graph.replay()
        torch.cuda.synchronize()
        for i, s in enumerate(seqs):
            m.tokens[s] = m.read(s)
            assert m.tokens[s].shape[2] == at[i] + 1 + step and np.isfinite(m.tokens[s]).all()
        got = out.clone()
        m.check(seqs, [1] * 3, [q_out])
        again = torch.empty_like(out)
        m.batch.attention_device(0, q_out, again)
        assert torch.equal(got, again)                        # the eager call gives the same bits
    assert m.batch.info()["reallocations"] == 0


def test_two_batches_over_one_cache_and_stale_plans(env):
    sat, torch, ctx = env
    m = Model(env, "f32", 64, 1, 2, 16, layers=1, seed=30)
    a, b, c = m.new(), m.new(), m.new()
    m.step([a, b, c], [20, 30, 40])
    other = sat.DecodeBatch(m.cache, 2)
    q = m.step([a, b], [1, 1])
    other.step([c], [1])                                      # another sequence: the first plan stands
    m.check([a, b], [1, 1], q)
    m.cache.extend([b], [1])
    out = torch.empty_like(q[0])
    with pytest.raises(sat.ArgumentError, match="changed"):
        m.batch.attention_device(0, q[0], out)
    m.cache.free([c])
    with pytest.raises(sat.ArgumentError, match="changed"):
        other.append_device(0, m.normal(1, 64), m.normal(1, 64))


def test_step_on_another_stream(env):
    sat, torch, ctx = env
    stream = torch.cuda.Stream()
    mine = sat.Context(0)
    mine.set_stream(stream.cuda_stream)
    m = Model((sat, torch, mine), "bf16", 64, 2, 2, 16, layers=1, seed=31)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        s = m.new()
        m.step([s], [50])
        q = m.step([s], [1])
        m.check([s], [1], q)
    del m
    mine.close()


def test_device_refusals(env):
    sat, torch, ctx = env
    m = Model(env, "bf16", 64, 2, 2, 16, layers=2)
    q = torch.zeros((1, 256), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((1, 128), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    with pytest.raises(sat.ArgumentError):
        m.batch.attention_device(0, q[:0], out[:0])           # no step yet
    s = m.new()
    m.batch.step([s], [1])
    for call in (lambda: m.batch.attention_device(2, q, out), lambda: m.batch.attention_device(-1, q, out),
                 lambda: m.batch.attention_device(0, q.float(), out), lambda: m.batch.attention_device(0, q, out.half()),
                 lambda: m.batch.attention_device(0, q.cpu(), out), lambda: m.batch.attention_device(0, q[:, ::2], out),
                 lambda: m.batch.attention_device(0, torch.cat([q, q]), out),
                 lambda: m.batch.append_device(0, k, k.float()), lambda: m.batch.append_device(0, k.half(), k.half()),
                 lambda: m.batch.append_device(0, k, k, q), lambda: m.batch.append_device(0, k, k, q, out.float()),
                 lambda: m.batch.append_device(0, k[:, :64], k), lambda: m.batch.append_device(5, k, k)):
        with pytest.raises(sat.ArgumentError):
            call()
    wide = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    m.batch.append_device(0, k, k, q, out)                    # and what fits is taken
    m.batch.step([s], [2])
    m.batch.attention_device(0, wide, torch.empty_like(wide))
    m.batch.step([s], [0])                                    # a step without rows does nothing
    m.batch.attention_device(0, q[:0], out[:0])
    with pytest.raises(sat.ArgumentError):
        sat.PagedCache(1, 4, 16, 1, 64, memory=torch.zeros(4 * 2 * 16 * 64 - 1, device="cuda"), ctx=ctx)
    with pytest.raises(sat.ArgumentError):
        sat.PagedCache(1, 4, 16, 1, 64, memory=torch.zeros(4 * 2 * 16 * 64).half(), ctx=ctx)
    own = sat.PagedCache(1, 4, 16, 1, 64, ctx=ctx)            # memory of its own
    assert own.info()["memory"] and own.info()["bytes"] == 4 * 2 * 16 * 64 * 4
    own.dispose()
    host = sat.PagedCache(1, 4, 16, 1, 64, ctx=False)
    with pytest.raises(sat.NotSupportedError):
        b = sat.DecodeBatch(host, 1)
        b.step(host.create(1), [1])
        b.attention_device(0, q, out)


def test_random_serving_run(env):
    """Requests come, fork, run behind shared prompts, rewind and leave while the cache is compacted."""
    sat, torch, ctx = env
    for kind, dim in (("bf16", 128), ("f32", 64), ("f16", 96)):
        m = Model(env, kind, dim, 2, 4, 32, pages=200, layers=2, rope=1e5, seed=dim)
        rng = np.random.default_rng(dim)
        root = m.new()
        m.step([root], [500])
        live = [root]
        for step in range(12):
            parent = int(rng.choice(live))
            live += m.fork([parent], [int(rng.integers(1, m.tokens[parent].shape[2] + 1))])
            if step % 3 == 2:
                s = live[int(rng.integers(len(live)))]
                at = int(rng.integers(1, m.tokens[s].shape[2] + 1))
                m.cache.rewind([s], [at])
                m.tokens[s] = m.tokens[s][:, :, :at]
            if len(live) > 6:
                gone = live.pop(0)
                m.cache.free([gone])
                m.cache.compact()
            order = [int(s) for s in rng.permutation(live)]
            counts = [int(rng.choice([1, 1, 1, 0, 25])) for _ in order]
            q = m.step(order, counts)
            m.check(order, counts, q)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,kv_heads,group,page", [(128, 2, 4, 32), (64, 2, 1, 64), (64, 1, 7, 16), (96, 1, 3, 16), (128, 1, 1, 128)])
@pytest.mark.parametrize("before,count", [(0, 2), (0, 70), (61, 9), (200, 300)])
def test_infinities_and_nan_in_masked_places(env, kind, dim, kv_heads, group, page, before, count):
    """What a token's K and V hold reaches the rows of the same step from that token on and no others: each column of
    the output takes the infinities and NaN of that column of the V it sees."""
    torch = env[1]
    m = Model(env, kind, dim, kv_heads, group, page, pages=64)
    s, other = m.new(), m.new()
    if before:
        m.step([s, other], [before, 3])
    counts = [count, 4]
    queries = m.step([s, other], counts)
    total = before + count
    inf = math.inf
    # (token, head, column, value); the second token's weight is above zero: scores are small.
    marks = [(before + 1, 0, 3, inf), (total - 1, 0, 3, -inf), (before + count // 2, kv_heads - 1, dim - 1, math.nan),
             (before + max(1, count // 3), 0, 40, -inf), (total - 1, kv_heads - 1, 17, math.nan)]
    table = m.cache.table(s)
    held = {(t, h, c): v for t, h, c, v in marks}      # (a later mark of the same place replaces it)
    for (t, h, c), v in held.items():
        m.pool[0, int(table[t // page]), 1, h, t % page, c] = v
    m.pool[1, int(table[(total - 1) // page]), 0, 0, (total - 1) % page, 5] = math.nan     # a key: its own row only
    keys, values = m.tokens[s][0].copy(), m.tokens[s][1].copy()
    for layer, q in enumerate(queries):
        out = torch.full((sum(counts), kv_heads * group * dim), 7.0, dtype=torch.float32, device="cuda")
        m.batch.attention_device(layer, q, out)
        got = out.double().cpu().numpy().reshape(-1, kv_heads, group, dim)
        qd = q.double().cpu().numpy().reshape(-1, kv_heads, group, dim)
        assert np.isfinite(got[count:]).all()
        for r in range(count):
            t = before + r + 1
            exact, size, scores = m.formula(qd[r], keys[layer, :t], values[layer, :t])
            special = np.zeros((kv_heads, dim))
            if layer == 0:
                with np.errstate(invalid="ignore"):
                    for (at, h, c), v in held.items():
                        if at < t:
                            special[h, c] += v
            elif r == count - 1:
                special[0] = math.nan
            special = np.broadcast_to(special[:, None], got[r].shape)
            strange = ~np.isfinite(special)
            assert np.array_equal(got[r][strange], special[strange], equal_nan=True), (layer, r)
            tol = (2 * (dim + 4) * scores[..., None] + 2 * (t + 16)) * U * size
            if kind != "f32":
                tol = tol + torch.finfo(m.dtype).eps / 2 * size
            assert np.all(np.abs(got[r] - exact)[~strange] <= tol[~strange]), (layer, r)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 4, 7), (64, 8, 1), (64, 2, 24), (128, 1, 25)])
@pytest.mark.parametrize("n,prefix,own", [(64, 1536, 1), (64, 1536, 130), (200, 0, 1), (150, 0, 64), (40, 260, 70)])
def test_many_short_segments_behind_long_ones(env, kind, dim, kv_heads, group, n, prefix, own):
    """Launches whose CTAs work through many one-block items between tiles of a shared prefix, run again and again:
    every run ends, with the same bits, and a sample of the rows is checked."""
    torch = env[1]
    page = 64
    m = Model(env, kind, dim, kv_heads, group, page, pages=-(-prefix // page) + n * (own // page + 2) + 8, layers=1)
    m.pool.copy_(m.normal(*m.pool.shape).to(m.dtype))         # contents enough: nothing is appended here
    if prefix:
        root = m.cache.create(1)
        m.cache.extend(root, [prefix])
        seqs = m.cache.fork(root * n)
    else:
        seqs = m.cache.create(n)
    if own > 1:
        m.cache.extend(seqs, [own - 1 - i % min(own - 1, 50) for i in range(n)])
    m.batch.step(seqs, [1] * n)
    q = m.normal(n, kv_heads * group * dim).to(m.dtype)
    out = torch.empty_like(q)
    m.batch.attention_device(0, q, out)
    torch.cuda.synchronize()
    for _ in range(30):
        again = torch.empty_like(q)
        m.batch.attention_device(0, q, again)
        assert torch.equal(out, again)
    rows = list(range(0, n, 13))
    for s in rows:
        m.tokens[seqs[s]] = m.read(seqs[s])
    qd, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    half = torch.finfo(m.dtype).eps / 2
    for s in rows:
        k, v = m.tokens[seqs[s]][:, 0]
        exact, size, scores = m.formula(qd[s].reshape(kv_heads, group, dim), k, v)
        tol = (2 * (dim + 4) * scores[..., None] + 2 * (len(k) + 16)) * U * size
        if kind != "f32":
            tol = tol + half * size + half * np.abs(exact) + torch.finfo(m.dtype).smallest_normal * half * 2
        assert np.all(np.abs(got[s].reshape(exact.shape) - exact) <= tol), s


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,kv_heads,group", [(16, 2, 3), (40, 1, 8), (80, 2, 1), (104, 2, 5), (120, 1, 12), (136, 2, 4)])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_heads_of_any_size(env, kind, dim, kv_heads, group, page):
    """Heads whose rows are no whole number of 128 bytes: single tokens, prompts and a shared prefix."""
    m = Model(env, kind, dim, kv_heads, group, page, layers=2, rope=1e4 if dim % 16 == 0 else 0.0, seed=dim)
    root = m.new()
    m.step([root], [300])
    seqs = m.fork([root] * 3, [300, 290, 70]) + [m.new()]
    counts = [1, 2, 90, 60]
    m.check(seqs, counts, m.step(seqs, counts))
    q = m.step(seqs, [1] * 4)
    m.check(seqs, [1] * 4, q, out_f32=True)
    m.check(seqs, [1] * 4, q, strided=True)


def test_rows_that_overlap(env):
    """Slices of the same wide rows are taken, rows that share values refused; a packed q may be rotated in place."""
    sat, torch, ctx = env
    m = Model(env, "bf16", 64, 2, 2, 16, layers=1, rope=1e4, seed=33)
    s = m.new()
    (q,) = m.step([s], [5])
    wide = torch.zeros((5, 512), dtype=torch.bfloat16, device="cuda")
    wide[:, :256] = q
    m.batch.attention_device(0, wide[:, :256], wide[:, 256:])
    out = torch.empty_like(q)
    m.batch.attention_device(0, q, out)
    assert torch.equal(wide[:, 256:], out) and torch.equal(wide[:, :256], q)
    flat = torch.zeros(4 * 5 * 256, dtype=torch.bfloat16, device="cuda")
    cut = lambda at: flat[at:at + 5 * 256].view(5, 256)
    for a, b in ((q, q), (wide[:, :256], wide[:, 128:384]), (wide[:, 128:384], wide[:, :256]), (cut(0), cut(255)),
                 (cut(5 * 256 - 1), cut(0)), (cut(8), flat[:5 * 512].view(5, 512)[:, 256:])):
        with pytest.raises(sat.ArgumentError, match="overlap"):
            m.batch.attention_device(0, a, b)
    m.batch.attention_device(0, cut(0), cut(5 * 256))         # neighbours
    k = m.normal(5, 128).to(torch.bfloat16)
    raw = m.normal(5, 256).to(torch.bfloat16)
    m.batch.append_device(0, k, k, raw, out)
    place = raw.clone()
    m.batch.append_device(0, k, k, place, place)
    assert torch.equal(place, out)
    fused = m.normal(5, 512).to(torch.bfloat16)
    with pytest.raises(sat.ArgumentError, match="overlap"):
        m.batch.append_device(0, fused[:, 256:384], fused[:, 384:], fused[:, :256], fused.view(-1)[:5 * 256].view(5, 256))
    with pytest.raises(sat.ArgumentError, match="overlap"):
        m.batch.append_device(0, k, k, cut(0), cut(64))
    with pytest.raises(sat.ArgumentError, match="overlap"):
        m.batch.append_device(0, cut(0)[:, :128], k, raw, cut(0))


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_of_one_batch(env, kind):
    """Each layer captured in a graph of its own: they share the plan and the space for partial results, and may be
    replayed in any order on one stream, between eager calls too."""
    sat, torch, ctx = env
    m = Model(env, kind, 64, 2, 4, 16, pages=128, layers=2, seed=40)
    root = m.new()
    m.step([root], [300])
    seqs = m.fork([root] * 3, [300, 290, 17])
    m.step(seqs, [1, 40, 130])
    queries = m.step(seqs, [1] * 3)
    q = [x.clone() for x in queries]
    out = [torch.zeros_like(x) for x in q]
    stream, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        for layer in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                m.batch.attention_device(layer, q[layer], out[layer])
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    for step in range(3):
        if step:
            queries = m.step(seqs, [1] * 3)
            for mine, new in zip(q, queries):
                mine.copy_(new)
        eager = [torch.empty_like(x) for x in q]
        for layer in (0, 1):
            m.batch.attention_device(layer, q[layer], eager[layer])
        for order in ((0, 1), (1, 0), (1, 1, 0)):
            for x in out:
                x.zero_()
            for layer in order:
                graphs[layer].replay()
                m.batch.attention_device(1 - layer, q[1 - layer], eager[1 - layer])
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
        m.check(seqs, [1] * 3, queries)
