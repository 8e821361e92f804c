"""Low-rank adapters of many requests beside a shared projection, against the 64-bit formula.

Tolerance: weights are exact; x and t = A x enter their products cut to 24 bits (2^-24 relative each, two
dropped products of 2^-24 more); the FP32 sums of n products are in error by at most n 2^-23 of the sum of
magnitudes (tensor cores may truncate: a whole step per addition).  With T = |A| |x| and O = |B| T:
|err| <= scale (cols 2^-23 + rank 2^-23 + 16 2^-24) O + 2 2^-24 (|base| + |out|).
"""
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


def _load(torch, aset, kind, rows, cols, ranks, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    got = []
    for slot, rank in enumerate(ranks):
        if rank == 0:
            got.append(None)
            continue
        a = (torch.randn((rank, cols), generator=g, device="cuda") / cols ** 0.5).to(_dtype(torch, kind))
        b = torch.randn((rows, rank), generator=g, device="cuda").to(_dtype(torch, kind))
        scale = 0.5 + slot
        aset.load(slot, a, b, scale)
        got.append((a.double(), b.double(), scale))
    return got


def _check(torch, out, x, base, ids, weights):
    rows, cols = out.shape[1], x.shape[1]
    exact, mag = base.double().clone(), torch.zeros_like(base, dtype=torch.float64)
    n = torch.zeros(len(ids), 1, dtype=torch.float64, device="cuda")
    for slot, w in enumerate(weights):
        at = torch.from_numpy(np.flatnonzero(np.asarray(ids) == slot)).cuda()
        if w is None or at.numel() == 0:
            continue
        a, b, scale = w
        xd = x[at].double()
        exact[at] += scale * (xd @ a.T) @ b.T
        mag[at] = scale * (xd.abs() @ a.abs().T) @ b.abs().T
        n[at] = 2.0 * (cols + a.shape[0]) + 16
    tol = n * U * mag + 2 * U * (base.abs().double() + exact.abs())
    err = (out.double() - exact).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    none = torch.from_numpy(np.asarray(ids) < 0).cuda()
    assert torch.equal(out[none], base[none])


KINDS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,ranks,n", [
    (64, 32, [16], 1), (1, 1, [1], 1), (777, 1000, [8, 3, 0, 16], 50), (3584, 1536, [16, 8], 8),
    (512, 3584, [64, 4, 33, 17, 50], 129), (96, 100, [128, 100, 1], 40), (1000, 31, [30, 32], 33),
    (18944, 256, [64], 17), (33, 8960, [20], 300)])
def test_formula(env, kind, rows, cols, ranks, n):
    sat, torch, ctx = env
    rng = np.random.default_rng(rows + n)
    aset = sat.AdapterSet(rows, cols, len(ranks), max(ranks), dtype=kind, ctx=ctx)
    weights = _load(torch, aset, kind, rows, cols, ranks, seed=cols)
    plan = sat.AdapterRows(ctx)
    g = torch.Generator(device="cuda").manual_seed(n)
    for ids in (rng.integers(-1, len(ranks), n), np.zeros(n, int), np.full(n, -1), np.arange(n) % len(ranks)):
        plan.assign(ids)
        x = torch.randn((n, cols), generator=g, device="cuda")
        base = torch.randn((n, rows), generator=g, device="cuda")
        out = torch.full_like(base, float("nan"))
        aset.apply_device(plan, x, base, out)
        _check(torch, out, x, base, ids, weights)
        inplace = base.clone()
        aset.apply_device(plan, x, inplace, inplace)
        assert torch.equal(inplace, out)


def test_strided_rows(env):
    sat, torch, ctx = env
    rows, cols, n = 70, 48, 21
    aset = sat.AdapterSet(rows, cols, 2, 16, dtype="bf16", ctx=ctx)
    weights = _load(torch, aset, "bf16", rows, cols, [16, 5])
    plan = sat.AdapterRows(ctx)
    ids = np.arange(n) % 3 - 1
    plan.assign(ids)
    for ox, ob, oo in ((0, 0, 0), (1, 2, 3), (4, 4, 4)):
        x = torch.randn((n, cols + 9), device="cuda")[:, ox:ox + cols]
        base = torch.randn((n, rows + 7), device="cuda")[:, ob:ob + rows]
        big = torch.full((n, rows + 8), 3.0, device="cuda")
        out = big[:, oo:oo + rows]
        aset.apply_device(plan, x, base, out)
        _check(torch, out, x, base, ids, weights)
        assert bool((big[:, :oo] == 3).all()) and bool((big[:, oo + rows:] == 3).all())


def test_slots_change_and_rows_beyond_keep_their_values(env):
    sat, torch, ctx = env
    aset = sat.AdapterSet(40, 64, 3, 32, dtype="f16", ctx=ctx)
    weights = _load(torch, aset, "f16", 40, 64, [32, 16, 7])
    plan = sat.AdapterRows(ctx)
    plan.assign([0, 1, 2, 0])
    x, base = torch.randn((6, 64), device="cuda"), torch.randn((6, 40), device="cuda")
    out = torch.full((6, 40), 9.0, device="cuda")
    aset.apply_device(plan, x[:4], base[:4], out[:4])
    _check(torch, out[:4], x[:4], base[:4], [0, 1, 2, 0], weights)
    assert bool((out[4:] == 9).all())
    aset.unload(1)
    host = np.random.default_rng(0).standard_normal((2, 64)).astype(np.float16)
    hb = np.random.default_rng(1).standard_normal((40, 2)).astype(np.float16)
    aset.load(0, host, hb, -1.5)                              # a smaller adapter in the place of a larger one
    weights[0] = (torch.from_numpy(host).cuda().double(), torch.from_numpy(hb).cuda().double(), -1.5)
    weights[1] = None
    aset.apply_device(plan, x[:4], base[:4], out[:4])
    exact = base[:4].double()
    for p, s in ((0, 0), (2, 2), (3, 0)):
        a, b, scale = weights[s]
        exact[p] += scale * b @ (a @ x[p].double())
    assert torch.allclose(out[:4].double(), exact, rtol=1e-5, atol=1e-5)     # 64 2^-23 of magnitudes below 100
    assert torch.equal(out[1], base[1])


def test_repeatable_bits_and_replay(env):
    """The same call gives the same bits; a captured call replays for the next assignment."""
    sat, torch, ctx = env
    rows, cols, n = 200, 96, 24
    aset = sat.AdapterSet(rows, cols, 4, 16, dtype="bf16", ctx=ctx)
    weights = _load(torch, aset, "bf16", rows, cols, [16, 8, 16, 2])
    plan = sat.AdapterRows(ctx)
    rng = np.random.default_rng(2)
    x, base = torch.randn((n, cols), device="cuda"), torch.randn((n, rows), device="cuda")
    out = torch.zeros_like(base)
    plan.assign([0] * n)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            aset.apply_device(plan, x, base, out)
            with pytest.raises(sat.NotSupportedError):
                plan.assign([0])
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    for _ in range(5):
        ids = rng.integers(-1, 4, n)
        plan.assign(ids)
        graph.replay()
        _check(torch, out, x, base, ids, weights)
        eager = torch.empty_like(out)
        aset.apply_device(plan, x, base, eager)
        again = torch.empty_like(out)
        aset.apply_device(plan, x, base, again)
        assert torch.equal(eager, again)


@pytest.mark.parametrize("fmt,order", [("Q4_0", "batch"), ("Q8_0", "batch"), ("Q4_0", "tensor")])
def test_beside_the_shared_projection(env, fmt, order):
    """execute_device = the quantized projection (its own bits) with the adapters of each row added."""
    sat, torch, ctx = env
    from satori_b200 import _lib
    rows, cols, n = 320, 256, 37
    f = getattr(sat, fmt)
    w = torch.randn(rows * cols, device="cuda") * 0.05
    payload = torch.empty(rows * (cols // 32) * (34 if f == sat.Q8_0 else 18), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().satori_quantize_q_device(ctx.handle, w.data_ptr(), rows, cols, f, payload.data_ptr()))
    m = sat.CudaQuantizedMatrix.from_device(ctx, payload.data_ptr(), payload.numel(), rows, cols, f)
    aset = sat.AdapterSet(rows, cols, 3, 16, ctx=ctx)
    weights = _load(torch, aset, "bf16", rows, cols, [16, 4, 9])
    plan = sat.AdapterRows(ctx)
    ids = np.arange(n) % 4 - 1
    plan.assign(ids)
    x = torch.randn((n, cols), device="cuda")
    base, out = torch.empty((n, rows), device="cuda"), torch.empty((n, rows), device="cuda")
    code = {"batch": _lib.ORDER_BATCH, "tensor": _lib.ORDER_TENSOR}[order]
    m.execute_device(x.data_ptr(), base.data_ptr(), n, code)
    aset.execute_device(m, plan, x, out, code)
    _check(torch, out, x, base, ids, weights)
    with pytest.raises(sat.ArgumentError):
        aset.execute_device(m, plan, x, x.new_empty((n, rows)), 7)
    other = sat.AdapterSet(rows + 1, cols, 3, 16, ctx=ctx)
    with pytest.raises(sat.ArgumentError):
        other.execute_device(m, plan, x, torch.empty((n, rows + 1), device="cuda"))


def test_refusals(env):
    sat, torch, ctx = env
    for bad in ((0, 8, 1, 8), (8, 0, 1, 8), (8, 8, 0, 8), (8, 8, 1, 0), (8, 8, -1, 8)):
        with pytest.raises(sat.ArgumentError):
            sat.AdapterSet(*bad, ctx=ctx)
    with pytest.raises(sat.NotSupportedError):
        sat.AdapterSet(8, 8, 1, 129, ctx=ctx)
    aset = sat.AdapterSet(16, 8, 2, 8, dtype="f32", ctx=ctx)
    plan = sat.AdapterRows(ctx)
    x, base = torch.zeros((2, 8), device="cuda"), torch.zeros((2, 16), device="cuda")
    out = torch.empty_like(base)
    with pytest.raises(sat.ArgumentError):
        aset.apply_device(plan, x[:0], base[:0], out[:0])     # nothing assigned yet
    a, b = torch.zeros((4, 8), device="cuda"), torch.zeros((16, 4), device="cuda")
    for call in (lambda: aset.load(2, a, b), lambda: aset.load(-1, a, b), lambda: aset.load(0, a, b[:, :3]),
                 lambda: aset.load(0, a.half(), b.half()), lambda: aset.load(0, a, b, float("nan")),
                 lambda: aset.load(0, torch.zeros((17, 8), device="cuda"), torch.zeros((16, 17), device="cuda")),
                 lambda: plan.assign([-2]), lambda: plan.assign([0.5]), lambda: aset.unload(5)):
        with pytest.raises(sat.ArgumentError):
            call()
    plan.assign([0, 2])
    with pytest.raises(sat.ArgumentError):
        aset.apply_device(plan, x, base, out)                 # slot 2 of two
    plan.assign([0, 1])
    big = torch.zeros((3, 16), device="cuda")
    for call in (lambda: aset.apply_device(plan, x[:1], base, out), lambda: aset.apply_device(plan, x.half(), base, out),
                 lambda: aset.apply_device(plan, x, base, out.cpu()), lambda: aset.apply_device(plan, x, big[:2], big[1:]),
                 lambda: aset.apply_device(plan, big.view(6, 8)[:2], base, big[:2])):
        with pytest.raises(sat.ArgumentError):
            call()
    aset.apply_device(plan, x, base, out)                     # empty slots add nothing
    assert torch.equal(out, base)
    plan.assign([])
    aset.apply_device(plan, x[:0], base[:0], out[:0])
    aset.dispose()
    aset.dispose()
    with pytest.raises(sat.DisposedError):
        aset.unload(0)


def test_rows_that_overlap(env):
    """x, base and out may be slices of the same wide rows, and out base itself; anything else that overlaps is refused."""
    sat, torch, ctx = env
    rows, cols, n = 64, 96, 20
    aset = sat.AdapterSet(rows, cols, 2, 8, ctx=ctx)
    weights = _load(torch, aset, "bf16", rows, cols, [8, 5])
    plan, ids = sat.AdapterRows(ctx), [0, 1] * 10
    plan.assign(ids)
    wide = torch.randn((n, cols + 2 * rows), device="cuda")
    x, base, out = wide.split([cols, rows, rows], 1)
    kept = wide.clone()
    aset.apply_device(plan, x, base, out)
    _check(torch, out, x, base, ids, weights)
    assert torch.equal(wide[:, :cols + rows], kept[:, :cols + rows])
    alone = out.clone()
    aset.apply_device(plan, x, base, base)                    # in place
    assert torch.equal(base, alone)
    for b, o in ((base, x[:, :rows]), (base, wide[:, cols - 1:cols - 1 + rows]), (base, wide[:, cols + 1:cols + 1 + rows]),
                 (base, wide.view(-1)[cols:cols + n * rows].view(n, rows))):
        with pytest.raises(sat.ArgumentError, match="overlap"):
            aset.apply_device(plan, x, b, o)


@pytest.mark.parametrize("kind", KINDS)
def test_values_of_every_magnitude(env, kind):
    """Rows of x from 2^-100 to 2^100 (no product passes FP32's range), zero rows, and columns of very different size:
    each part that a value is cut into keeps 2^-22 of it, or 2^-39 of the largest beside it."""
    sat, torch, ctx = env
    rows, cols, n = 96, 200, 34
    aset = sat.AdapterSet(rows, cols, 2, 24, dtype=kind, ctx=ctx)
    weights = _load(torch, aset, kind, rows, cols, [24, 7], 3)
    plan, ids = sat.AdapterRows(ctx), np.arange(n) % 2
    plan.assign(ids)
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((n, cols), generator=g, device="cuda")
    x[:17] *= 2.0 ** torch.linspace(-100, 100, 17, device="cuda").round()[:, None]
    x[17] = 0
    x[18:26, ::3] *= 2.0 ** -20
    x[26:, :64] *= 2.0 ** 12
    base = torch.zeros((n, rows), device="cuda")
    out = torch.empty_like(base)
    aset.apply_device(plan, x, base, out)
    _check(torch, out, x, base, ids, weights)
    assert bool((out[17] == 0).all())
