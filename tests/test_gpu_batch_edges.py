"""Batch attention and adapters where one launch, replay or value meets another: strange keys that rows see, partial
records without a finite score, small weights, many merged rows, moved plans, launches that overlap.

Tolerances are those of test_gpu_batch.py where nothing else is said.
"""
import math

import numpy as np
import pytest

from test_gpu_batch import KINDS, U, Model, env  # noqa: F401  (env: the fixture)

pytestmark = pytest.mark.gpu


def _filled(env, kind, dim, kv_heads, group, page, pages, layers, seed):
    """A model whose pages all hold normal values: nothing has to be appended."""
    m = Model(env, kind, dim, kv_heads, group, page, pages=pages, layers=layers, seed=seed)
    m.pool.normal_(generator=m.torch.Generator(device="cuda").manual_seed(seed))
    return m


def _attend(m, layer, q, rows):
    out = m.torch.full((rows, m.kv * m.group * m.dim), 7.0, dtype=m.torch.float32, device="cuda")
    m.batch.attention_device(layer, q, out)
    return out.double().cpu().numpy().reshape(rows, m.kv, m.group, m.dim)


def _tolerance(m, t, exact, size, scores):
    tol = (2 * (m.dim + 4) * scores[..., None] + 2 * (t + 16)) * U * size
    return tol if m.kind == "f32" else tol + m.torch.finfo(m.dtype).eps / 2 * size


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,group,n,own", [(128, 8, 40, 1), (64, 8, 40, 1), (64, 1, 1, 200), (136, 8, 9, 1)])
@pytest.mark.parametrize("special", [math.nan, math.inf, -math.inf])
def test_a_strange_key_reaches_the_rows_that_see_it(env, kind, dim, group, n, own, special):  # noqa: F811
    """A key that every row sees, at each of a block's 64 places: a NaN or infinite score makes the row NaN, a score of
    minus infinity leaves the row without that key."""
    torch = env[1]
    m = _filled(env, kind, dim, 8, group, 64, 8 + 2 * n * (-(-own // 64)), 8, 5)
    root = m.cache.create(1)
    m.cache.extend(root, [256])
    seqs = m.cache.fork(root * n)
    m.batch.step(seqs, [own] * n)
    table = m.cache.table(seqs[0])
    for layer in range(8):
        for h in range(8):
            token = 64 + 8 * layer + h
            m.pool[layer, int(table[token // 64]), 0, h, token % 64, 3] = special
    rows = n * own
    q = m.normal(rows, 8 * group * dim).to(m.dtype).view(rows, -1, dim)
    q[..., 3] = q[..., 3].abs() + 0.5
    qd = q.double().cpu().numpy().reshape(rows, 8, group, dim)
    some = [s for s in (0, n // 2, n - 1)]
    tokens = {s: m.read(seqs[s]) for s in some}
    for layer in range(8):
        got = _attend(m, layer, q.view(rows, -1), rows)
        if special != -math.inf:
            assert np.isnan(got).all(), layer
            continue
        assert np.isfinite(got).all(), layer
        for s in some:
            for r in (0, own - 1):
                t = 256 + r + 1
                k, v = tokens[s][:, layer, :t]
                for h in range(8):
                    seen = np.arange(t) != 64 + 8 * layer + h
                    exact, size, scores = m.formula(qd[s * own + r, h:h + 1], k[seen][:, h:h + 1], v[seen][:, h:h + 1])
                    err = np.abs(got[s * own + r, h:h + 1] - exact)
                    assert np.all(err <= _tolerance(m, t, exact, size, scores)), (layer, s, r, h)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 136])
@pytest.mark.parametrize("special", [math.nan, math.inf])
def test_a_strange_key_in_a_row_without_partial_records(env, kind, dim, special):  # noqa: F811
    """Prompts of 200 rows, enough of them that most tiles are one item that writes the outputs itself."""
    n, own = 48, 200
    m = _filled(env, kind, dim, 8, 1, 64, 6 * n, 8, 10)
    seqs = m.cache.create(n)
    m.cache.extend(seqs, [64] * n)
    m.batch.step(seqs, [own] * n)
    first = m.torch.tensor([int(m.cache.table(s)[0]) for s in seqs], device="cuda")
    for layer in range(8):
        for h in range(8):
            m.pool[layer, first, 0, h, 8 * layer + h, 3] = special
    q = m.normal(n * own, 8, dim).to(m.dtype)
    q[..., 3] = q[..., 3].abs() + 0.5
    for layer in range(8):
        assert np.isnan(_attend(m, layer, q.view(n * own, -1), n * own)).all(), layer


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 136])
@pytest.mark.parametrize("n", [4, 520])
def test_a_nan_key_alone_in_its_record(env, kind, dim, n):  # noqa: F811
    """The only key of a partial record (a request's first own token behind a shared prefix) scores NaN: the merge must
    not take the record for an empty one."""
    m = _filled(env, kind, dim, 4, 2, 16, 16 + n, 1, 6)
    root = m.cache.create(1)
    m.cache.extend(root, [256])
    seqs = m.cache.fork(root * n)
    m.batch.step(seqs, [1] * n)
    assert m.batch.info()["segments"] == n + 1
    marked = list(range(0, n, 3))
    for s in marked:
        m.pool[0, int(m.cache.table(seqs[s])[16]), 0, s % 4, 0, 1] = math.nan
    q = m.normal(n, 8 * dim).to(m.dtype)
    got = _attend(m, 0, q, n)
    nan = np.zeros((n, 4), bool)
    nan[marked, [s % 4 for s in marked]] = True
    assert np.array_equal(np.isnan(got).all((2, 3)), nan) and np.isfinite(got[~nan]).all()


def test_small_weights_beside_fp16_pages(env):  # noqa: F811
    """8192 keys of weight 2^-26 beside one of weight 1: together they are 2^-13 of the row.  A weight is rounded to fp16
    from 2^7 times itself, so by at most 2^-12 of it or 2^-32 (half a subnormal step of 2^-24, over 2^7)."""
    torch = env[1]
    n, kv, dim = 37, 4, 64                                     # 148 tiles: an SM works through most of a row's keys
    m = Model(env, "f16", dim, kv, 4, 64, pages=n * 129, layers=1)
    seqs = m.cache.create(n)
    m.cache.extend(seqs, [8192] * n)
    m.batch.step(seqs, [1] * n)
    first_pages = [int(m.cache.table(s)[0]) for s in seqs]
    assert first_pages == [128 * i for i in range(n)]          # the last page of each lies behind all of these
    q = torch.zeros((n, kv * 4, dim), dtype=m.dtype, device="cuda")
    q[..., 0] = 26 * math.log(2) * 8
    weight = math.exp(-float(q[0, 0, 0]) / 8)
    exact = 8192 * weight / (1 + 8192 * weight)
    tol = 8192 * (2.0 ** -12 * weight + 2.0 ** -32) + (2 * 68 * 19 + 2 * 8209) * U * exact
    for heavy in (0, 5000, 8191):                              # where the heavy key lies
        m.pool[:, :, 0].zero_()
        m.pool[:, :, 1].fill_(1.0)
        pages = torch.tensor(first_pages, device="cuda") + heavy // 64
        m.pool[0, pages, 0, :, heavy % 64, 0] = 1.0
        m.pool[0, pages, 1, :, heavy % 64] = 0.0
        got = _attend(m, 0, q.view(n, -1), n)
        assert np.all(np.abs(got - exact) <= tol), (heavy, np.abs(got - exact).max(), tol)


def test_many_merged_rows_of_many_heads(env):  # noqa: F811
    """16000 rows of 32 KV heads behind a shared prefix: every row and head is merged."""
    torch = env[1]
    dim, kv, n, own = 128, 32, 64, 250
    m = _filled(env, "bf16", dim, kv, 1, 64, 8 + 4 * n, 1, 8)
    root = m.cache.create(1)
    m.cache.extend(root, [512])
    seqs = m.cache.fork(root * n)
    m.batch.step(seqs, [own] * n)
    q = m.normal(n * own, kv * dim).to(m.dtype)
    got = _attend(m, 0, q, n * own)
    for s in (0, 31, 63):
        k, v = m.read(seqs[s])[:, 0]
        for r in (0, 1, 100, 249):
            t = 512 + r + 1
            qd = q[s * own + r].double().cpu().numpy().reshape(kv, 1, dim)
            exact, size, scores = m.formula(qd, k[:t], v[:t])
            assert np.all(np.abs(got[s * own + r] - exact) <= _tolerance(m, t, exact, size, scores)), (s, r)


def test_a_replay_follows_an_assignment_that_outgrows_its_plan(env):  # noqa: F811
    sat, torch, ctx = env
    rows, cols, n = 16, 32, 20000
    aset = sat.AdapterSet(rows, cols, 2, 4, dtype="f32", ctx=ctx)
    g = torch.Generator(device="cuda").manual_seed(9)
    for slot in range(2):
        aset.load(slot, torch.randn((4, cols), generator=g, device="cuda"), torch.randn((rows, 4), generator=g, device="cuda"))
    plan = sat.AdapterRows(ctx)
    plan.assign([0, 1, -1])
    x, base = torch.randn((n, cols), generator=g, device="cuda"), torch.randn((n, rows), generator=g, device="cuda")
    out = torch.zeros_like(base)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            aset.apply_device(plan, x[:3], base[:3], out[:3])  # (the buffers behind hold 20000 rows)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    for ids in (np.arange(17000) % 3 - 1, np.arange(5) % 2, np.arange(n) % 2, np.full(9, -1)):
        plan.assign(ids)
        out.fill_(7.0)
        graph.replay()
        want = torch.full_like(out, 7.0)
        k = len(ids)
        aset.apply_device(plan, x[:k], base[:k], want[:k])
        # (The replay's clusters may be dealt differently from the eager call's: the sums' order is another.)
        assert torch.allclose(out, want, rtol=0, atol=1e-3) and torch.equal(out[k:], want[k:])


def _on_stream(torch, ctx, stream):
    """Routes the context to a stream for a while."""
    import contextlib

    @contextlib.contextmanager
    def scope():
        torch.cuda.synchronize()
        ctx.set_stream(stream.cuda_stream)
        try:
            yield
        finally:
            torch.cuda.synchronize()
            ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return scope()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 4, 7), (136, 2, 4)])
@pytest.mark.parametrize("behind", ["projection", "adapters", "attention"])
def test_outputs_without_a_merge_reach_the_launch_behind(env, request, kind, dim, kv_heads, group, behind):  # noqa: F811
    """Requests of at most 64 tokens: every item writes its outputs itself and the merge has no row.  The next launch
    may start early; it gets the attention's outputs all the same, eager and in a graph."""
    sat, torch, ctx = env
    n, width = 64, kv_heads * group * dim
    m = _filled(env, kind, dim, kv_heads, group, 16, 5 * n, 1, 11)
    seqs = m.cache.create(n)
    m.cache.extend(seqs, [10 + i % 53 for i in range(n)])
    m.batch.step(seqs, [1] * n)
    assert m.batch.info()["items"] == n * kv_heads
    q = m.normal(n, width).to(m.dtype)
    att = torch.zeros((n, width), dtype=m.dtype if behind == "attention" else torch.float32, device="cuda")
    if behind == "projection":
        from satori_b200 import _lib
        payload = torch.empty(256 * (width // 32) * 34, dtype=torch.uint8, device="cuda")
        w = m.normal(256 * width) * 0.05
        _lib.check(_lib.lib().satori_quantize_q_device(ctx.handle, w.data_ptr(), 256, width, sat.Q8_0, payload.data_ptr()))
        matrix = sat.CudaQuantizedMatrix.from_device(ctx, payload.data_ptr(), payload.numel(), 256, width, sat.Q8_0)
        request.addfinalizer(matrix.dispose)
        out = torch.zeros((1, 256), device="cuda")
        after = lambda: matrix.execute_device(att[n - 1].data_ptr(), out.data_ptr(), 1, _lib.ORDER_BATCH)
    elif behind == "adapters":
        aset = sat.AdapterSet(256, width, 2, 16, ctx=ctx)
        for slot in range(2):
            aset.load(slot, m.normal(16, width).bfloat16(), m.normal(256, 16).bfloat16())
        plan = sat.AdapterRows(ctx)
        plan.assign([i % 3 - 1 for i in range(n)])
        base, out = m.normal(n, 256), torch.zeros((n, 256), device="cuda")
        after = lambda: aset.apply_device(plan, att, base, out)
    else:
        out = torch.zeros((n, width), dtype=m.dtype, device="cuda")
        after = lambda: m.batch.attention_device(0, att, out)
    stream = torch.cuda.Stream()
    with _on_stream(torch, ctx, stream), torch.cuda.stream(stream):
        m.batch.attention_device(0, q, att)
        stream.synchronize()
        after()
        stream.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            m.batch.attention_device(0, q, att)
            after()
        for run in range(40):
            att.fill_(math.nan)
            out.fill_(math.nan)
            stream.synchronize()
            if run % 2:
                graph.replay()
            else:
                m.batch.attention_device(0, q, att)
                after()
            stream.synchronize()
            assert torch.equal(out, want), run


def test_an_application_without_items_waits_for_the_launch_before(env):  # noqa: F811
    """Replayed after an assignment of no rows between an attention and its reader."""
    sat, torch, ctx = env
    n = 64
    m = _filled(env, "bf16", 128, 4, 7, 16, 5 * n, 1, 12)
    seqs = m.cache.create(n)
    m.cache.extend(seqs, [10 + i % 53 for i in range(n)])
    m.batch.step(seqs, [1] * n)
    q = m.normal(n, 28 * 128).to(m.dtype)
    att = torch.zeros((n, 28 * 128), device="cuda")
    first, second = sat.AdapterRows(ctx), sat.AdapterRows(ctx)
    first.assign([0] * n)
    second.assign([0] * n)
    aset = sat.AdapterSet(96, 28 * 128, 1, 16, ctx=ctx)
    aset.load(0, m.normal(16, 28 * 128).bfloat16(), m.normal(96, 16).bfloat16())
    base, unused, out = m.normal(n, 96), torch.zeros((n, 96), device="cuda"), torch.zeros((n, 96), device="cuda")
    stream = torch.cuda.Stream()
    with _on_stream(torch, ctx, stream), torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            m.batch.attention_device(0, q, att)
            aset.apply_device(first, att, base, unused)
            aset.apply_device(second, att, base, out)
        graph.replay()
        stream.synchronize()
        want = out.clone()
        first.assign([])
        for _ in range(20):
            att.fill_(math.nan)
            out.fill_(math.nan)
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want)


def test_a_replay_with_a_slot_that_its_adapters_lack(env):  # noqa: F811
    """The call itself refuses such a slot; a replay after a later assignment leaves the row's base and reports it."""
    sat, torch, ctx = env
    aset = sat.AdapterSet(48, 64, 2, 8, dtype="f32", ctx=ctx)
    for slot in range(2):
        aset.load(slot, torch.randn((8, 64), device="cuda"), torch.randn((48, 8), device="cuda"))
    plan = sat.AdapterRows(ctx)
    plan.assign([0, 1, 0, -1])
    x, base = torch.randn((4, 64), device="cuda"), torch.randn((4, 48), device="cuda")
    out, want = torch.zeros_like(base), torch.zeros_like(base)
    stream = torch.cuda.Stream()
    with _on_stream(torch, ctx, stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            aset.apply_device(plan, x, base, out)
    plan.assign([1, -1, -1, 0])
    aset.apply_device(plan, x, base, want)
    ctx.synchronize()
    plan.assign([1, 2, 1 << 30, 0])
    with pytest.raises(sat.ArgumentError):
        aset.apply_device(plan, x, base, want)
    graph.replay()
    with pytest.raises(sat.ArgumentError, match="slot"):
        ctx.synchronize()
    assert torch.allclose(out, want, rtol=0, atol=1e-3)        # (the items differ, and with them the order of sums)
    assert torch.equal(out[1:3], base[1:3])
    plan.assign([1, -1, -1, 0])
    graph.replay()
    ctx.synchronize()                                          # reported once


def test_rows_of_another_context_are_refused(env, request):  # noqa: F811
    sat, torch, ctx = env
    other = sat.Context(0)
    try:
        aset = sat.AdapterSet(16, 32, 1, 4, dtype="f32", ctx=ctx)
        foreign = sat.AdapterRows(other)
        foreign.assign([0, -1])
        x, base = torch.zeros((2, 32), device="cuda"), torch.zeros((2, 16), device="cuda")
        with pytest.raises(sat.ArgumentError, match="context"):
            aset.apply_device(foreign, x, base, torch.zeros_like(base))
        payload = torch.zeros(16 * 34, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        matrix = sat.CudaQuantizedMatrix.from_device(ctx, payload.data_ptr(), payload.numel(), 16, 32, sat.Q8_0)
        request.addfinalizer(matrix.dispose)
        with pytest.raises(sat.ArgumentError, match="context"):
            aset.execute_device(matrix, foreign, x, torch.zeros_like(base))
        foreign.dispose()
    finally:
        other.close()


def test_transposed_weights_on_a_context_with_its_own_stream(env):  # noqa: F811
    """load makes a packed copy of a transposed tensor on torch's stream; the context's reads it only then."""
    sat, torch, _ = env
    mine = sat.Context(0)
    try:
        rows, cols = 64, 96
        aset = sat.AdapterSet(rows, cols, 1, 16, dtype="f32", ctx=mine)
        plan = sat.AdapterRows(mine)
        plan.assign([0] * 5)
        for seed in range(3):
            g = torch.Generator(device="cuda").manual_seed(seed)
            a, b = torch.randn((cols, 16), generator=g, device="cuda"), torch.randn((16, rows), generator=g, device="cuda")
            x, base = torch.randn((5, cols), generator=g, device="cuda"), torch.zeros((5, rows), device="cuda")
            out = torch.empty_like(base)
            torch.cuda.synchronize()
            torch.cuda._sleep(50_000_000)                      # torch's stream is busy for some 25 ms
            aset.load(0, a.T, b.T)
            aset.apply_device(plan, x, base, out)
            mine.synchronize()
            exact = (x.double() @ a.double()) @ b.double()
            assert torch.allclose(out.double(), exact, rtol=0, atol=(96 + 16 + 16) * 2 * U * float((x.abs() @ a.abs() @ b.abs()).max()))
        plan.dispose()
        aset.dispose()
    finally:
        mine.close()


def test_handles_of_a_closed_context(env):  # noqa: F811
    sat, torch, _ = env
    mine = sat.Context(0)
    cache = sat.PagedCache(1, 4, 16, 1, 64, ctx=mine)
    batch = sat.DecodeBatch(cache, 1)
    rows, aset = sat.AdapterRows(mine), sat.AdapterSet(8, 8, 1, 4, ctx=mine)
    s = cache.create(1)
    mine.close()
    for call in (lambda: cache.create(1), lambda: cache.fork(s), lambda: batch.step(s, [1]), lambda: rows.assign([0]),
                 lambda: aset.unload(0), lambda: cache.info()):
        with pytest.raises(sat.DisposedError):
            call()
    for handle in (batch, cache, rows, aset):
        handle.dispose()


def test_adapters_cannot_change_inside_a_capture(env):  # noqa: F811
    """The refusals leave the capture as it is."""
    sat, torch, ctx = env
    aset = sat.AdapterSet(16, 32, 2, 4, dtype="f32", ctx=ctx)
    a, b = torch.randn((4, 32), device="cuda"), torch.randn((16, 4), device="cuda")
    aset.load(0, a, b)
    plan = sat.AdapterRows(ctx)
    plan.assign([0, -1, 0])
    x, base = torch.randn((3, 32), device="cuda"), torch.randn((3, 16), device="cuda")
    out, want = torch.zeros_like(base), torch.zeros_like(base)
    aset.apply_device(plan, x, base, want)
    stream = torch.cuda.Stream()
    with _on_stream(torch, ctx, stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            aset.apply_device(plan, x, base, out)
            with pytest.raises(sat.NotSupportedError):
                aset.load(0, a, b)
            with pytest.raises(sat.NotSupportedError):
                aset.unload(0)
            with pytest.raises(sat.NotSupportedError):
                sat.AdapterSet(16, 32, 1, 4, ctx=ctx)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", ["Q8_0", "Q4_0"])
@pytest.mark.parametrize("rows,cols", [(512, 3584), (256, 1536), (1000, 18944), (33, 40000)])
def test_projections_of_several_rows_fit(env, request, fmt, rows, cols):  # noqa: F811
    """Narrow and long projections of a batch, whose positions or block sums do not all fit shared memory at once:
    every row has the bits that it has alone."""
    sat, torch, ctx = env
    from satori_b200 import _lib
    n, f = 11, getattr(sat, fmt)
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = torch.randn(rows * cols, generator=g, device="cuda") * 0.05
    payload = torch.empty(rows * (cols // 32) * (34 if f == sat.Q8_0 else 18), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().satori_quantize_q_device(ctx.handle, w.data_ptr(), rows, cols, f, payload.data_ptr()))
    matrix = sat.CudaQuantizedMatrix.from_device(ctx, payload.data_ptr(), payload.numel(), rows, cols, f)
    request.addfinalizer(matrix.dispose)
    x = torch.randn((n, cols), generator=g, device="cuda")
    alone, together, adapted = (torch.full((n, rows), math.nan, device="cuda") for _ in range(3))
    for p in range(n):
        matrix.execute_device(x[p].data_ptr(), alone[p].data_ptr(), 1)
    matrix.execute_device(x.data_ptr(), together.data_ptr(), n)
    assert torch.equal(together, alone)
    aset, plan = sat.AdapterSet(rows, cols, 1, 4, ctx=ctx), sat.AdapterRows(ctx)
    plan.assign([-1, 0] * 5 + [-1])                           # an empty slot adds nothing either
    aset.execute_device(matrix, plan, x, adapted)
    assert torch.equal(adapted, alone)
