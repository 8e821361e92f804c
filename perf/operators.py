"""The operators that decode many requests from one paged cache, as measured cases.

Four operators: the cache's pages (fork, copy, free, compact), the append of a batch's new tokens, the batch's
attention with shared prefixes computed once, and the low-rank adapters of many requests beside a shared
projection.  ``run`` computes a case in elementary torch operations when ``own`` is false and through
``satori_b200`` when it is true.  Sizes are those of the model shapes this repository carries (28 query / 4 KV
heads of 128, 3584 -> 3584 / 18944; 12 / 2 heads, 1536 -> 8960), or generic ones.
"""
import heapq
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROPE_BASE = 1e6


# ---------------------------------------------------------------- cases
def listed():
    return [
        # A beam step of one request: eight beams forked from a prompt of 300 tokens, half of them dropped.
        {"name": "pages_beam8", "op": "pages", "type": "bf16", "layers": 4, "kv_heads": 4, "dim": 128, "page": 16,
         "prompt": 300, "children": 8, "extend": 5},
        # 64 answers sampled from one 8k prompt over all layers of the 28-layer shape, half of them finished.
        {"name": "pages_fork64", "op": "pages", "type": "bf16", "layers": 28, "kv_heads": 4, "dim": 128, "page": 64,
         "prompt": 8229, "children": 64, "extend": 256},
        # One decode step of 64 requests: FP32 projections into a bf16 cache.
        {"name": "append_decode64", "op": "append", "type": "bf16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 16,
         "seqs": 64, "rows": 1, "context": 2000},
        # A prompt chunk of eight requests into an FP32 cache.
        {"name": "append_prompt", "op": "append", "type": "f32", "heads": 28, "kv_heads": 4, "dim": 128, "page": 64,
         "seqs": 8, "rows": 511, "context": 700},
        # The smallest step: one request, one token, a short FP32 cache.
        {"name": "attn_single", "op": "attention", "type": "f32", "heads": 28, "kv_heads": 4, "dim": 128, "page": 16,
         "seqs": 1, "rows": 1, "prefix": 0, "private": 300},
        # Sixteen unrelated requests of ragged lengths around 4k.
        {"name": "attn_private16", "op": "attention", "type": "bf16", "heads": 28, "kv_heads": 4, "dim": 128,
         "page": 16, "seqs": 16, "rows": 1, "prefix": 0, "private": 4096},
        # 64 requests behind one 32k document.
        {"name": "attn_prefix32k", "op": "attention", "type": "bf16", "heads": 28, "kv_heads": 4, "dim": 128,
         "page": 64, "seqs": 64, "rows": 1, "prefix": 32768, "private": 700},
        # Sixteen requests behind an 8k prompt in the framework's FP32 cache, 12 / 2 heads.
        {"name": "attn_prefix8k_f32", "op": "attention", "type": "f32", "heads": 12, "kv_heads": 2, "dim": 128,
         "page": 32, "seqs": 16, "rows": 1, "prefix": 8192, "private": 200},
        # The prompts of eight requests behind a shared 4k instruction, heads of 64.
        {"name": "attn_prompt_f16", "op": "attention", "type": "f16", "heads": 16, "kv_heads": 4, "dim": 64,
         "page": 32, "seqs": 8, "rows": 500, "prefix": 4096, "private": 500},
        # One decode step of eight requests with four adapters on a square projection.
        {"name": "lora_decode8", "op": "adapters", "type": "bf16", "columns": 3584, "out": 3584, "rows": 8, "slots": 4,
         "rank": 16},
        # A full batch with many adapters of mixed ranks on the gate projection.
        {"name": "lora_decode128", "op": "adapters", "type": "f16", "columns": 3584, "out": 18944, "rows": 128,
         "slots": 32, "rank": 64},
        # A prompt chunk of a few requests on the smaller shape's gate projection.
        {"name": "lora_prompt", "op": "adapters", "type": "bf16", "columns": 1536, "out": 8960, "rows": 4000,
         "slots": 3, "rank": 64},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["pages", "append", "attention", "attention", "attention", "adapters", "adapters"])
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    heads, kv_heads, dim = rng.choice([(28, 4, 128), (12, 2, 128), (8, 8, 64), (16, 4, 64), (6, 1, 128), (10, 2, 96)])
    page = rng.choice([16, 32, 64, 128])
    if op == "pages":
        return {"op": op, "type": kind, "layers": rng.randint(1, 12), "kv_heads": kv_heads, "dim": dim, "page": page,
                "prompt": _log(rng, 1, 6000), "children": _log(rng, 1, 40), "extend": _log(rng, 1, 200)}
    if op == "append":
        rows = rng.choice([1, 1, _log(rng, 1, 500)])
        return {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "seqs": _log(rng, 1, 64) if rows == 1 else rng.randint(1, 7), "rows": rows,
                "context": _log(rng, 1, 4000)}
    if op == "attention":
        rows = rng.choice([1, 1, 1, _log(rng, 2, 300)])
        seqs = _log(rng, 1, 60) if rows == 1 else rng.randint(1, 8)
        private = max(rows, _log(rng, 1, 3000 if rows == 1 else 500))
        return {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": seqs,
                "rows": rows, "prefix": rng.choice([0, _log(rng, 16, 16000 if rows == 1 else 3500)]),
                "private": private}
    shape = rng.choice([(3584, 3584), (3584, 512), (1536, 8960), (3584, 18944), (1000, 777)])
    rows = _log(rng, 1, 3000 if shape[1] < 10000 else 200)
    return {"op": op, "type": kind, "columns": shape[0], "out": shape[1], "rows": rows,
            "slots": rng.randint(1, 24 if rows < 256 else 4), "rank": rng.choice([4, 8, 16, 24, 32, 64])}


def _fixed(case):
    """The ragged sizes of a case: the same for every seed."""
    return np.random.RandomState(sum(v * k for k, v in enumerate(
        (v for _, v in sorted(case.items()) if isinstance(v, int)), 17)) % (1 << 31))


def _ragged(case, key, n, least=1):
    """n sizes between half of case[key] and all of it; the first is all of it."""
    top = case[key]
    low = max(least, top // 2)
    sizes = _fixed(case).randint(low, max(low, top) + 1, n)
    sizes[0] = max(top, least)
    return [int(v) for v in sizes]


# ---------------------------------------------------------------- page bookkeeping of the plain form
class Pages:
    """Sequences as lists of page numbers; the lowest free page is taken first."""

    def __init__(self, pages, page):
        self.page, self.count, self.live, self.heap = page, pages, {}, list(range(pages))

    def take(self):
        p = heapq.heappop(self.heap)
        self.live[p] = 1
        return p

    def extend(self, seq, n):
        seq["length"] += n
        seq["pages"] += [self.take() for _ in range(-(-seq["length"] // self.page) - len(seq["pages"]))]

    def fork(self, seq, position):
        whole = position // self.page
        child = {"pages": seq["pages"][:whole], "length": position}
        for p in child["pages"]:
            self.live[p] += 1
        pair = []
        if position % self.page:
            child["pages"].append(self.take())
            pair = [(seq["pages"][whole], child["pages"][whole])]
        return child, pair

    def free(self, seq):
        for p in seq["pages"]:
            self.live[p] -= 1
            if not self.live[p]:
                del self.live[p]
                heapq.heappush(self.heap, p)

    def compact(self, seqs):
        n = len(self.live)
        moves = list(zip(sorted(p for p in self.live if p >= n), sorted(p for p in self.heap if p < n)))
        to = dict(moves)
        self.live = {to.get(p, p): c for p, c in self.live.items()}
        self.heap = list(range(n, self.count))
        for s in seqs:
            s["pages"] = [to.get(p, p) for p in s["pages"]]
        return moves


def _pages_plan(case):
    """(pages needed, fork positions, extensions)."""
    n = case["children"]
    r = _fixed(case)
    positions = [int(v) for v in r.randint(max(1, case["prompt"] - 2 * case["page"]), case["prompt"] + 1, n)]
    extra = [int(v) for v in r.randint(max(1, case["extend"] // 2), case["extend"] + 1, n)]
    need = -(-case["prompt"] // case["page"]) + sum(-(-e // case["page"]) + 1 for e in extra)
    return need, positions, extra


def _pages_moves(pages, parent, positions, extra):
    """One pass on the bookkeeping: the fork's copies, the compaction's moves, and the surviving tables."""
    forked = [pages.fork(parent, p) for p in positions]
    children = [c for c, _ in forked]
    for c, e in zip(children, extra):
        pages.extend(c, e)
    for c in children[1::2]:
        pages.free(c)
    kept = children[0::2]
    moves = pages.compact(kept + [parent])
    tables = [list(c["pages"]) for c in kept]
    for c in kept:
        pages.free(c)
    return [p for _, pair in forked for p in pair], moves, tables


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _context():
    import satori_b200 as sat
    ctx = sat.default_context(torch.cuda.current_device())
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream by its handle
    return sat, ctx


def _layout(case):
    """Where the tokens of a batch lie, the lowest free page first: (prefix pages, [private pages], private lengths,
    pages in all).  Every request starts behind the prefix's whole pages; its private tokens follow them."""
    page, prefix = case["page"], case.get("prefix", 0)
    whole = prefix // page
    tail = prefix - whole * page
    lengths = _ragged(case, "private", case["seqs"], case["rows"]) if "private" in case else \
        [c + n for c, n in zip(_ragged(case, "context", case["seqs"]), _counts(case))]
    at = whole + (1 if tail else 0)
    shared = list(range(whole))
    private = [[] for _ in lengths]
    if tail:  # every fork copies the prefix's partial page first
        private = [[at + b] for b in range(len(lengths))]
        at += len(lengths)
    for b, n in enumerate(lengths):
        more = -(-(tail + n) // page) - len(private[b])
        private[b] += list(range(at, at + more))
        at += more
    return shared, private, [tail + n for n in lengths], at


def _counts(case):
    return _ragged(case, "rows", case["seqs"]) if case["rows"] > 1 else [1] * case["seqs"]


def _row_index(counts):
    """Row -> (sequence, place among the sequence's rows)."""
    seq = np.repeat(np.arange(len(counts)), counts)
    place = np.concatenate([np.arange(n) for n in counts])
    return seq, place


def _pool(case, layers, pages, seed):
    shape = (layers, pages, 2, case["kv_heads"], case["page"], case["dim"])
    return torch.randn(shape, generator=_generator(seed), device="cuda", dtype=TYPES[case["type"]])


def _prepare_pages(case, seed):
    need, positions, extra = _pages_plan(case)
    pages = Pages(need, case["page"])
    parent = {"pages": [], "length": 0}
    pages.extend(parent, case["prompt"])
    s = {"case": case, "pool": _pool(case, case["layers"], need, seed), "pages": pages, "parent": parent,
         "positions": positions, "extra": extra}
    if own:
        sat, ctx = _context()
        s["cache"] = sat.PagedCache(case["layers"], need, case["page"], case["kv_heads"], case["dim"],
                                    dtype=case["type"], memory=s["pool"], ctx=ctx)
        s["root"] = s["cache"].create(1)
        s["cache"].extend(s["root"], [case["prompt"]])
    return s


def _prepare_batch(case, seed):
    shared, private, lengths, pages = _layout(case)
    pool = _pool(case, 1, pages, seed)
    counts = _counts(case)
    seq, place = _row_index(counts)
    prefix = len(shared) * case["page"]
    before = np.array(lengths) - np.array(counts) + prefix        # cached tokens before the step
    positions = before[seq] + place
    s = {"case": case, "pool": pool, "counts": counts}
    table = np.zeros((len(private), max(map(len, private))), np.int64)
    for b, p in enumerate(private):
        table[b, :len(p)] = p
    s["shared"] = torch.tensor(shared, dtype=torch.int64, device="cuda")
    s["table"] = torch.from_numpy(table).cuda()
    s["seq"], s["place"] = torch.from_numpy(seq).cuda(), torch.from_numpy(place).cuda()
    s["limit"] = torch.from_numpy(positions - prefix + 1).cuda()  # private tokens that a row may read
    s["positions"] = torch.from_numpy(positions).cuda()
    tail = case.get("prefix", 0) - prefix
    if tail:  # the forks' copies of the prefix's partial page
        pool[:, s["table"][:, 0], :, :, :tail] = pool[:, len(shared):len(shared) + 1, :, :, :tail]
    if own:
        sat, ctx = _context()
        cache = sat.PagedCache(1, pages, case["page"], case["kv_heads"], case["dim"], dtype=case["type"],
                               memory=pool, ctx=ctx)
        if case.get("prefix", 0):
            root = cache.create(1)
            cache.extend(root, [case["prefix"]])
            # A fork copies the prefix's partial page whole, over the tokens behind it that lie there already.
            kept = pool[:, s["table"][:, 0]].clone()
            seqs = cache.fork(root * len(counts))
            torch.cuda.synchronize()
            pool[:, s["table"][:, 0]] = kept
        else:
            seqs = cache.create(len(counts))
        # Each sequence's pages follow one another: all of its tokens get room, then the step's go again.
        cache.extend(seqs, [int(a) + n - cache.length(q) for a, n, q in zip(before, counts, seqs)])
        cache.rewind(seqs, [int(a) for a in before])
        batch = sat.DecodeBatch(cache, case["heads"], rope_base=ROPE_BASE)
        batch.step(seqs, counts)
        s["cache"], s["batch"] = cache, batch
    return s


def _prepare_append(case, seed):
    s = _prepare_batch(case, seed)
    n, heads, kv, dim = sum(s["counts"]), case["heads"], case["kv_heads"], case["dim"]
    s["qkv"] = torch.randn((n, (heads + 2 * kv) * dim), generator=_generator(seed + 1), device="cuda")
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    angle = s["positions"].double()[:, None] / torch.pow(torch.tensor(ROPE_BASE, dtype=torch.float64, device="cuda"),
                                                          2 * i / dim)
    s["cos"], s["sin"] = angle.cos(), angle.sin()  # one table for all layers of a step
    s["q_out"] = torch.empty((n, heads * dim), dtype=TYPES[case["type"]], device="cuda")
    return s


def _prepare_attention(case, seed):
    s = _prepare_batch(case, seed)
    n, kind = sum(s["counts"]), TYPES[case["type"]]
    s["q"] = torch.randn((n, case["heads"] * case["dim"]), generator=_generator(seed + 1), device="cuda", dtype=kind)
    s["out"] = torch.empty_like(s["q"])
    return s


def _adapter_ranks(case):
    """Ranks of the slots: the case's rank and smaller ones."""
    return [int(v) for v in np.maximum(1, case["rank"] // np.array([1, 2, 1, 4])[np.arange(case["slots"]) % 4])]


def _adapter_rows(case):
    """The slot of each row: runs of the same request's rows; every ninth run has no adapter (-1)."""
    r = _fixed(case)
    n, got = case["rows"], []
    run = max(1, n // (2 * case["slots"]))
    while len(got) < n:
        slot = -1 if len(got) and r.randint(9) == 0 else int(r.randint(case["slots"]))
        got += [slot] * int(r.randint(1, run + 1))
    return np.array(got[:n], np.int32)


def _prepare_adapters(case, seed):
    g, kind = _generator(seed), TYPES[case["type"]]
    k, m, r, slots = case["columns"], case["out"], case["rank"], case["slots"]
    s = {"case": case, "ids": _adapter_rows(case)}
    s["x"] = torch.randn((case["rows"], k), generator=g, device="cuda")
    s["base"] = torch.randn((case["rows"], m), generator=g, device="cuda")
    keep = torch.arange(r, device="cuda")[None, :] < torch.tensor(_adapter_ranks(case), device="cuda")[:, None]
    s["a"] = torch.randn((slots, r, k), generator=g, device="cuda", dtype=kind) / math.sqrt(k) * keep[:, :, None].to(kind)
    s["b"] = torch.randn((slots, m, r), generator=g, device="cuda", dtype=kind) * keep[:, None, :].to(kind)
    s["scale"] = [2.0 / (1 + v % 3) for v in range(slots)]
    slot = torch.from_numpy(s["ids"].astype(np.int64)).cuda()
    s["pick"] = (slot[:, None] == torch.arange(slots, device="cuda")[None, :]).float() * \
        torch.tensor(s["scale"], device="cuda")[None, :]
    s["out"] = torch.empty_like(s["base"])
    if own:
        sat, ctx = _context()
        s["set"] = sat.AdapterSet(m, k, slots, r, dtype=case["type"], ctx=ctx)
        for v, rank in enumerate(_adapter_ranks(case)):
            s["set"].load(v, s["a"][v, :rank], s["b"][v, :, :rank], s["scale"][v])
        s["plan"] = sat.AdapterRows(ctx)
        s["plan"].assign(s["ids"])
    return s


def prepare(case, seed):
    return {"pages": _prepare_pages, "append": _prepare_append, "attention": _prepare_attention,
            "adapters": _prepare_adapters}[case["op"]](case, seed)


# ---------------------------------------------------------------- one pass
def _padded(tables):
    out = np.full((len(tables), max(map(len, tables))), -1, np.int32)
    for i, t in enumerate(tables):
        out[i, :len(t)] = t
    return out


def _run_pages(s):
    pool = s["pool"]
    if own:
        cache = s["cache"]
        children = cache.fork(s["root"] * len(s["positions"]), s["positions"])
        cache.extend(children, s["extra"])
        cache.free(children[1::2])
        moved = cache.compact()
        tables = [cache.table(c) for c in children[0::2]]
        cache.free(children[0::2])
        return {"pool": pool, "tables": _padded(tables), "moved": moved}
    copies, moves, tables = _pages_moves(s["pages"], s["parent"], s["positions"], s["extra"])
    for pairs in (copies, moves):
        if pairs:
            src, dst = torch.tensor(pairs, device="cuda").unbind(1)
            pool[:, dst] = pool[:, src]
    return {"pool": pool, "tables": _padded(tables), "moved": len(moves)}


def _rotated(x, cos, sin, half):
    """RopeHalf on [rows, heads, dim]: pairs (i, i + half)."""
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * cos[:, None] - b * sin[:, None], a * sin[:, None] + b * cos[:, None]], -1)


def _run_append(s):
    c = s["case"]
    heads, kv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    q, k, v = s["qkv"].split([heads * dim, kv * dim, kv * dim], 1)
    if own:
        s["batch"].append_device(0, k, v, q, s["q_out"])
        return {"q": s["q_out"], "pool": s["pool"]}
    kind, n = s["pool"].dtype, q.shape[0]
    at = s["limit"] - 1
    where = s["table"][s["seq"], at // page]
    pool = s["pool"][0]
    pool[where, 0, :, at % page] = _rotated(k.view(n, kv, dim), s["cos"], s["sin"], dim // 2).to(kind)
    pool[where, 1, :, at % page] = v.reshape(n, kv, dim).to(kind)
    s["q_out"][:] = _rotated(q.view(n, heads, dim), s["cos"], s["sin"], dim // 2).view(n, -1).to(kind)
    return {"q": s["q_out"], "pool": s["pool"]}


def _run_attention(s):
    if own:
        s["batch"].attention_device(0, s["q"], s["out"])
        return s["out"]
    c = s["case"]
    kv, dim, group = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    pool, seqs, rows = s["pool"][0], len(s["counts"]), max(s["counts"])
    q = torch.zeros((seqs, rows, c["heads"] * dim), device="cuda")
    q[s["seq"], s["place"]] = s["q"].float()
    q = q.view(seqs, rows, kv, group, dim).permute(2, 0, 3, 1, 4) / math.sqrt(dim)       # [kv, seqs, group, rows, dim]
    limit = torch.ones((seqs, rows), dtype=torch.int64, device="cuda")
    limit[s["seq"], s["place"]] = s["limit"]
    # The shared prefix once for all rows, then each sequence's own tokens under its causal limit.
    tokens = len(s["shared"]) * c["page"]
    kp, vp = pool[s["shared"]].float().permute(1, 2, 0, 3, 4).reshape(2, kv, tokens, dim)
    first = (q.reshape(kv, -1, dim) @ kp.transpose(1, 2)).view(kv, seqs, group, rows, tokens)
    own_kv = pool[s["table"]].float().permute(2, 3, 0, 1, 4, 5).reshape(2, kv, seqs, -1, dim)
    then = (q.reshape(kv, seqs, -1, dim) @ own_kv[0].transpose(2, 3)).view(kv, seqs, group, rows, -1)
    hidden = torch.arange(then.shape[-1], device="cuda") >= limit[:, None, :, None]
    then.masked_fill_(hidden, float("-inf"))
    top = then.amax(-1, keepdim=True)
    if tokens:
        top = torch.maximum(top, first.amax(-1, keepdim=True))
    first, then = (first - top).exp_(), (then - top).exp_()
    total = first.sum(-1, keepdim=True) + then.sum(-1, keepdim=True)
    # Values behind a sequence's end weigh nothing whatever they are.
    value = own_kv[1].masked_fill(torch.arange(own_kv.shape[3], device="cuda")[:, None] >=
                                  limit.amax(1)[:, None, None], 0.0)
    out = (first.reshape(kv, seqs * group * rows, tokens) @ vp).view(kv, seqs, group, rows, dim)
    out = out + (then.reshape(kv, seqs, group * rows, -1) @ value).view(kv, seqs, group, rows, dim)
    out = (out / total).permute(1, 3, 0, 2, 4).reshape(seqs, rows, -1)
    s["out"][:] = out[s["seq"], s["place"]].to(s["out"].dtype)
    return s["out"]


def _run_adapters(s):
    if own:
        s["set"].apply_device(s["plan"], s["x"], s["base"], s["out"])
        return s["out"]
    slots, r, k = s["a"].shape
    t = (s["x"] @ s["a"].float().view(-1, k).T).view(-1, slots, r) * s["pick"][:, :, None]
    b = s["b"].float().permute(0, 2, 1).reshape(slots * r, -1)
    s["out"][:] = s["base"] + t.view(-1, slots * r) @ b
    return s["out"]


def run(state):
    return {"pages": _run_pages, "append": _run_append, "attention": _run_attention,
            "adapters": _run_adapters}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "pages":
        need, positions, extra = _pages_plan(case)
        pages = Pages(need, case["page"])
        parent = {"pages": [], "length": 0}
        pages.extend(parent, case["prompt"])
        copies, moves, _ = _pages_moves(pages, parent, positions, extra)
        return {"bytes": 2 * (len(copies) + len(moves)) * case["layers"] * 2 * case["kv_heads"] * case["page"] *
                case["dim"] * size, "flops": 0}
    if case["op"] == "adapters":
        ids, ranks = _adapter_rows(case), _adapter_ranks(case)
        k, m = case["columns"], case["out"]
        used = sum(ranks[v] for v in set(ids.tolist()) if v >= 0)
        per_row = sum(ranks[v] for v in ids.tolist() if v >= 0)
        return {"bytes": case["rows"] * (k + 2 * m) * 4 + used * (k + m) * size, "flops": 2 * per_row * (k + m)}
    counts = _counts(case)
    n, heads, kv, dim = sum(counts), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        return {"bytes": n * (heads + 2 * kv) * dim * (4 + size), "flops": 3 * n * (heads + kv) * dim}
    shared, _, lengths, _ = _layout(case)
    prefix = len(shared) * case["page"]
    visible = sum(c * (prefix + n - c) + c * (c + 1) // 2 for c, n in zip(counts, lengths))
    return {"bytes": (prefix + sum(lengths)) * 2 * kv * dim * size + 2 * n * heads * dim * size,
            "flops": 4 * heads * dim * visible}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_append(case, s):
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows = s["qkv"].double().view(-1, heads + 2 * kv, dim)
    half = dim // 2
    pool, turned = s["pool"].double(), torch.empty_like(rows)
    turned.copy_(rows)
    position = s["positions"].double()
    for i in range(half):
        angle = position * ROPE_BASE ** (-2.0 * i / dim)
        c, z = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        a, b = rows[:, :heads + kv, i], rows[:, :heads + kv, i + half]
        turned[:, :heads + kv, i] = c * a - z * b
        turned[:, :heads + kv, i + half] = z * a + c * b
    at = s["limit"] - 1
    where = s["table"][s["seq"], at // page]
    pool[0][where, 0, :, at % page] = turned[:, heads:heads + kv]
    pool[0][where, 1, :, at % page] = turned[:, heads + kv:]
    return {"q": turned[:, :heads].reshape(rows.shape[0], -1), "pool": pool}


def _exact_attention(case, s):
    kv, dim, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    answers, row = [], 0
    shared, private, lengths, _ = _layout(case)
    for pages, length, count in zip(private, lengths, s["counts"]):
        held = s["pool"][0][torch.tensor(shared + pages, device="cuda")].double()       # [pages, 2, kv, page, dim]
        keys, values = (held[:, j].permute(1, 0, 2, 3).reshape(kv, -1, dim) for j in (0, 1))
        n = len(shared) * case["page"] + length
        keys, values = keys[:, :n], values[:, :n]
        q = s["q"][row:row + count].double().view(count, kv, group, dim)
        part = torch.empty_like(q)
        step = max(1, int(2e8 // (group * n)))
        for h in range(kv):
            for a in range(0, count, step):
                some = q[a:a + step, h]
                score = torch.einsum("rgd,td->rgt", some, keys[h]) / dim ** 0.5
                last = n - count + 1 + torch.arange(a, a + some.shape[0], device="cuda")
                score[(torch.arange(n, device="cuda")[None, :] >= last[:, None])[:, None].expand_as(score)] = -torch.inf
                part[a:a + step, h] = torch.softmax(score, -1) @ values[h]
        answers.append(part.reshape(count, -1))
        row += count
    return torch.cat(answers)


def _exact_adapters(case, s):
    out = s["base"].double()
    for v in range(case["slots"]):
        rows = torch.from_numpy(np.flatnonzero(s["ids"] == v)).cuda()
        if rows.numel():
            low = s["x"][rows].double() @ s["a"][v].double().T
            out[rows] += s["scale"][v] * (low @ s["b"][v].double().T)
    return out


def exact(case, seed):
    if case["op"] == "pages":
        return None  # copies and page numbers: nothing is computed
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "adapters": _exact_adapters}[case["op"]](case, s)
