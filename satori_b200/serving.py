"""Decoding many requests together: a paged key/value cache and the batch that steps over it.

The reference decodes one sequence per session (``DenseSession``); this module mirrors the part of the C ABI
that a host needs to serve many: ``PagedCache`` (sequences as lists of pages, forked without copying their
full pages), ``DecodeBatch`` (append and grouped attention for the new tokens of several sequences; keys that
sequences share are read once), ``AdapterSet`` and ``AdapterRows`` (the low-rank adapters of each row's
request beside a shared projection).  Device vectors are torch CUDA tensors, or any object with ``data_ptr``,
``dtype``, ``shape`` and ``stride``; the work is queued on the context's stream.
"""
from __future__ import annotations

import ctypes as C
from array import array

import numpy as np

from . import _lib
from ._lib import ArgumentError, DisposedError, check
from .core import Context, CudaQuantizedMatrix, default_context

_vp = C.c_void_p

_TYPES = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}
_TORCH_TYPES = {"torch.float32": _lib.F32, "torch.float16": _lib.F16, "torch.bfloat16": _lib.BF16}


def _bad(message: str) -> ArgumentError:
    return ArgumentError(_lib.ERR_ARGUMENT, message)


def _open(ctx) -> bool:
    """A handle whose context has been closed cannot be used or destroyed any more: its memory went with the
    process's use of the context."""
    return ctx is None or bool(ctx._h)


def _live(h, ctx, what: str):
    """The handle, while it and its context are open."""
    if not h:
        raise DisposedError(_lib.ERR_DISPOSED, f"{what} disposed")
    if not _open(ctx):
        raise DisposedError(_lib.ERR_DISPOSED, "context is disposed")
    return h


def _type(dtype) -> int:
    """'f32' / 'f16' / 'bf16', a torch dtype, or a satori_type."""
    t = _TYPES.get(dtype, _TORCH_TYPES.get(str(dtype), dtype))
    if t not in (_lib.F32, _lib.F16, _lib.BF16):
        raise _bad(f"unsupported type {dtype!r}")
    return t


_kinds: dict = {}                                             # torch dtype -> satori_type or None


def _kind(dtype):
    try:
        return _kinds[dtype]
    except KeyError:
        kind = _kinds[dtype] = _TORCH_TYPES.get(str(dtype))
        return kind


class _Ints:
    """Integers as a C int array: `size`, `address`, and what owns the memory."""
    __slots__ = ("size", "address", "owner")

    def __init__(self, values, name: str):
        if isinstance(values, (list, tuple, range)):
            try:
                self.owner = a = array("i", values)
            except TypeError:
                raise _bad(f"{name} must be a list of integers") from None
            except OverflowError:
                raise _bad(f"{name} exceeds Int32 limits") from None
            self.address, self.size = a.buffer_info()
            return
        a = np.asarray(values)
        if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
            raise _bad(f"{name} must be a list of integers")
        if a.size and (a.min() < -0x80000000 or a.max() > 0x7FFFFFFF):
            raise _bad(f"{name} exceeds Int32 limits")
        self.owner = a = np.ascontiguousarray(a, np.int32)
        self.address, self.size = a.ctypes.data, a.size


def _new_ints(n: int) -> tuple:
    """(array, address) of n integers to be filled in."""
    a = array("i", bytes(4 * n))
    return a, a.buffer_info()[0]


def _rows(t, rows: int, width: int, name: str, device: int, types) -> tuple:
    """(address, row stride, satori_type) of a device matrix of `rows` rows of `width` values."""
    kind = _kind(t.dtype)
    if kind is None or kind not in types:
        raise _bad(f"{name} has type {t.dtype}")
    if t.get_device() != device:
        raise _bad(f"{name} is not on device {device}")
    shape, stride = t.shape, t.stride()
    if len(shape) == 2 and shape[0] == rows and shape[1] == width and stride[1] == 1:
        ld = stride[0] if rows > 1 else width
    else:
        # Trailing dimensions are one packed row.
        n, at, packed = 1, len(shape), True
        while at > 1:
            at -= 1
            packed = packed and (shape[at] == 1 or stride[at] == n)
            n *= shape[at]
        if len(shape) == 0 or shape[0] != rows or n != width or not packed:
            raise _bad(f"{name} must be {rows} rows of {width} packed values, got shape {tuple(shape)} with strides {stride}")
        ld = stride[0] if rows > 1 else width
    if ld < width:
        raise _bad(f"{name}: rows overlap (row stride {ld})")
    return t.data_ptr(), ld, kind


class PagedCache:
    """Keys and values of many sequences in `pages` pages of `page_tokens` tokens, laid out
    [layer][page][K, V][kv_head][token][head_dim].  `memory`: a contiguous CUDA tensor of that many elements to
    use (kept alive here); None allocates.  ``ctx=False`` keeps the tables only (no device memory)."""

    def __init__(self, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, dtype="f32", memory=None,
                 ctx: Context | None = None):
        self._h = _vp()
        self.ctx = None if ctx is False else ctx or default_context()
        self.type = _type(dtype)
        self.layers, self.pages, self.page_tokens = layers, pages, page_tokens
        self.kv_heads, self.head_dim = kv_heads, head_dim
        address = None
        if memory is not None:
            if self.ctx is None:
                raise _bad("memory without a context")
            if _kind(memory.dtype) != self.type:
                raise _bad(f"memory has type {memory.dtype}")
            if not memory.is_cuda or memory.device.index != self.ctx.device or not memory.is_contiguous():
                raise _bad("memory must be a contiguous tensor on the context's device")
            if memory.numel() != layers * pages * 2 * kv_heads * page_tokens * head_dim:
                raise _bad("memory does not match the cache's shape")
            address = memory.data_ptr()
        self.memory = memory
        self._count = C.c_int()
        self._count_ref = C.byref(self._count)
        self._grow_scratch(1024)
        h = _vp()
        check(_lib.lib().satori_pages_create(self.ctx.handle if self.ctx else None, layers, pages, page_tokens, kv_heads,
                                             head_dim, self.type, address, C.byref(h)), "pages_create")
        self._h = h

    @property
    def handle(self):
        return _live(self._h, self.ctx, "paged cache is")

    def create(self, n: int = 1) -> list:
        """Ids of n new empty sequences."""
        if n < 0:
            raise _bad("n must not be negative")
        ids, address = _new_ints(n)
        check(_lib.lib().satori_pages_new(self.handle, n, address), "pages_new")
        return ids.tolist()

    def extend(self, seqs, counts) -> None:
        """Room for counts[i] more (unwritten) tokens at the end of each sequence."""
        s, c = self._pair(seqs, counts, "counts")
        check(_lib.lib().satori_pages_extend(self.handle, s.size, s.address, c.address), "pages_extend")

    def fork(self, parents, positions=None) -> list:
        """New sequences that share the parents' first positions[i] tokens (default: all of them)."""
        return self._fork(parents, positions, 1)

    def copy(self, parents, positions=None) -> list:
        """New sequences with pages of their own that hold the parents' first positions[i] tokens."""
        return self._fork(parents, positions, 0)

    def _fork(self, parents, positions, share: int) -> list:
        if positions is None:
            s, at = _Ints(parents, "parents"), None
        else:
            s, at = self._pair(parents, positions, "positions")
        ids, address = _new_ints(s.size)
        check(_lib.lib().satori_pages_fork(self.handle, s.size, s.address, at.address if at is not None else None, share,
                                           address), "pages_fork")
        return ids.tolist()

    def rewind(self, seqs, positions) -> None:
        """Discards the tokens at and after positions[i]."""
        s, at = self._pair(seqs, positions, "positions")
        check(_lib.lib().satori_pages_rewind(self.handle, s.size, s.address, at.address), "pages_rewind")

    def free(self, seqs) -> None:
        s = _Ints(seqs, "seqs")
        check(_lib.lib().satori_pages_free(self.handle, s.size, s.address), "pages_free")

    def compact(self) -> int:
        """Moves the live pages to the lowest numbers; the number of pages moved."""
        moved = C.c_int()
        check(_lib.lib().satori_pages_compact(self.handle, C.byref(moved)), "pages_compact")
        return moved.value

    def table(self, seq: int) -> np.ndarray:
        """The sequence's page numbers."""
        check(_lib.lib().satori_pages_table(self.handle, seq, None, self._scratch_at, self._scratch_size, self._count_ref),
              "pages_table")
        n = self._count.value
        if n > self._scratch_size:
            self._grow_scratch(2 * n)
            return self.table(seq)
        return self._scratch[:n].copy()

    def _grow_scratch(self, n: int) -> None:
        self._scratch = np.empty(n, np.int32)
        self._scratch_at, self._scratch_size = self._scratch.ctypes.data, n

    def length(self, seq: int) -> int:
        """The sequence's tokens."""
        length = C.c_int()
        check(_lib.lib().satori_pages_table(self.handle, seq, C.byref(length), None, 0, None), "pages_table")
        return length.value

    def copies(self) -> np.ndarray:
        """The [n, 2] (from, to) page pairs that the last fork, copy, rewind or compact copied."""
        count = C.c_int()
        check(_lib.lib().satori_pages_copies(self.handle, None, 0, C.byref(count)), "pages_copies")
        pairs = np.empty((count.value, 2), np.int32)
        check(_lib.lib().satori_pages_copies(self.handle, pairs.ctypes.data, count.value, None), "pages_copies")
        return pairs

    def info(self) -> dict:
        used, free, top, nbytes, memory = C.c_int(), C.c_int(), C.c_int(), C.c_size_t(), _vp()
        check(_lib.lib().satori_pages_info(self.handle, C.byref(used), C.byref(free), C.byref(top), C.byref(nbytes),
                                           C.byref(memory)), "pages_info")
        return {"used": used.value, "free": free.value, "top": top.value, "bytes": nbytes.value,
                "memory": memory.value or 0}

    @staticmethod
    def _pair(seqs, values, name: str) -> tuple:
        s, v = _Ints(seqs, "seqs"), _Ints(values, name)
        if s.size != v.size:
            raise _bad(f"{s.size} sequences, {v.size} {name}")
        return s, v

    def dispose(self) -> None:
        if self._h:
            if _open(self.ctx):
                _lib.lib().satori_pages_destroy(self._h)
            self._h = _vp()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass


class DecodeBatch:
    """The sequences of a paged cache that take a step together.  ``step`` extends them by their new tokens
    and plans the work once; ``append_device`` and ``attention_device`` then run for each layer."""

    def __init__(self, cache: PagedCache, q_heads: int, rope_base: float = 0.0, rotary: int = 0):
        self._h = _vp()
        self.cache = cache
        h = _vp()
        check(_lib.lib().satori_batch_create(cache.handle, q_heads, float(rope_base), rotary, C.byref(h)), "batch_create")
        self._h = h
        self.q_width, self.kv_width = q_heads * cache.head_dim, cache.kv_heads * cache.head_dim
        self.rows = 0

    @property
    def handle(self):
        return _live(self._h, self.cache.ctx, "batch is")

    def step(self, seqs, counts) -> None:
        """Extends each sequence by counts[i] new tokens; the step's rows are these tokens in order."""
        s, c = PagedCache._pair(seqs, counts, "counts")
        check(_lib.lib().satori_batch_step(self.handle, s.size, s.address, c.address), "batch_step")
        self.rows = int(sum(c.owner))

    def append_device(self, layer: int, k, v, q=None, q_out=None) -> None:
        """k and v (rows x kv_heads * head_dim; k is rotated) into the layer's pages; q rotated into q_out.
        Inputs are all float32 or all of the cache's type; rows may be strided (slices of fused rows)."""
        t, device = self.cache.type, self._device()
        kp, ldk, kind = _rows(k, self.rows, self.kv_width, "k", device, (_lib.F32, t))
        vp, ldv, kind_v = _rows(v, self.rows, self.kv_width, "v", device, (kind,))
        qp, ldq, op = None, 0, None
        if (q is None) != (q_out is None):
            raise _bad("q and q_out come together")
        if q is not None:
            qp, ldq, _ = _rows(q, self.rows, self.q_width, "q", device, (kind,))
            op, ldo, _ = _rows(q_out, self.rows, self.q_width, "q_out", device, (t,))
            if ldo != self.q_width:
                raise _bad("q_out must be packed")
        check(_lib.lib().satori_batch_append_device(self.handle, layer, kind, qp, ldq, kp, ldk, vp, ldv, op),
              "batch_append")

    def attention_device(self, layer: int, q, out) -> None:
        """Grouped attention of every row over its sequence up to its own position; q has the cache's type,
        out the cache's type or float32."""
        t, device = self.cache.type, self._device()
        qp, ldq, _ = _rows(q, self.rows, self.q_width, "q", device, (t,))
        op, ldo, kind = _rows(out, self.rows, self.q_width, "out", device, (t, _lib.F32))
        check(_lib.lib().satori_batch_attention_device(self.handle, layer, qp, ldq, op, ldo, kind), "batch_attention")

    def info(self) -> dict:
        rows, segments, items, moved = C.c_int(), C.c_int(), C.c_int(), C.c_int()
        check(_lib.lib().satori_batch_info(self.handle, C.byref(rows), C.byref(segments), C.byref(items),
                                           C.byref(moved)), "batch_info")
        return {"rows": rows.value, "segments": segments.value, "items": items.value, "reallocations": moved.value}

    def _device(self) -> int:
        if self.cache.ctx is None:
            raise _lib.NotSupportedError(_lib.ERR_NOT_SUPPORTED, "the cache has no device memory")
        return self.cache.ctx.device

    def dispose(self) -> None:
        if self._h:
            if _open(self.cache.ctx):
                _lib.lib().satori_batch_destroy(self._h)
            self._h = _vp()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass


class AdapterRows:
    """Which adapter slot each row of a batch uses (-1: none), for all projections of a step; for adapter sets of the
    same context."""

    def __init__(self, ctx: Context | None = None):
        self._h = _vp()
        self.ctx = ctx or default_context()
        h = _vp()
        check(_lib.lib().satori_adapter_rows_create(self.ctx.handle, C.byref(h)), "adapter_rows_create")
        self._h = h
        self.rows = 0

    @property
    def handle(self):
        return _live(self._h, self.ctx, "adapter rows are")

    def assign(self, slots) -> None:
        s = _Ints(slots, "slots")
        check(_lib.lib().satori_adapter_rows_assign(self.handle, s.size, s.address), "adapter_rows_assign")
        self.rows = s.size

    def dispose(self) -> None:
        if self._h:
            if _open(self.ctx):
                _lib.lib().satori_adapter_rows_destroy(self._h)
            self._h = _vp()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass


class AdapterSet:
    """The low-rank adapters of one projection of `rows` x `columns`: slot s adds
    scale * B (A x) with A [rank, columns] and B [rows, rank]."""

    def __init__(self, rows: int, columns: int, slots: int, max_rank: int, dtype="bf16", ctx: Context | None = None):
        self._h = _vp()
        self.ctx = ctx or default_context()
        self.type = _type(dtype)
        h = _vp()
        check(_lib.lib().satori_adapters_create(self.ctx.handle, rows, columns, slots, max_rank, self.type, C.byref(h)),
              "adapters_create")
        self._h = h
        self.rows, self.columns, self.slots = rows, columns, slots

    @property
    def handle(self):
        return _live(self._h, self.ctx, "adapters are")

    def load(self, slot: int, a, b, scale: float = 1.0) -> None:
        """A [rank, columns] and B [rows, rank]: CUDA tensors or host arrays / CPU tensors of the set's type;
        rows may be strided."""
        rank = int(a.shape[0])
        if tuple(a.shape) != (rank, self.columns) or tuple(b.shape) != (self.rows, rank) or rank < 1:
            raise _bad(f"A {tuple(a.shape)} and B {tuple(b.shape)} do not fit {self.rows} x {self.columns}")
        (ap, lda, keep_a), (bp, ldb, keep_b) = self._weights(a, "A"), self._weights(b, "B")
        check(_lib.lib().satori_adapters_load(self.handle, slot, rank, ap, lda, bp, ldb, scale), "adapters_load")
        del keep_a, keep_b

    def unload(self, slot: int) -> None:
        """Empties a slot: its rows get their projection alone."""
        check(_lib.lib().satori_adapters_load(self.handle, slot, 0, None, 0, None, 0, 0.0), "adapters_unload")

    def _weights(self, w, name: str) -> tuple:
        """(address, row stride in elements, what to keep alive)."""
        if not hasattr(w, "data_ptr"):
            w = np.asarray(w)
            kinds = {"float32": _lib.F32, "float16": _lib.F16}
            if kinds.get(str(w.dtype)) != self.type:
                raise _bad(f"{name} has type {w.dtype}")
            w = np.ascontiguousarray(w)
            return w.ctypes.data, w.shape[1], w
        if _kind(w.dtype) != self.type:
            raise _bad(f"{name} has type {w.dtype}")
        if w.is_cuda and w.device.index != self.ctx.device:
            raise _bad(f"{name} is not on device {self.ctx.device}")
        if (w.shape[1] > 1 and w.stride(1) != 1) or (w.shape[0] > 1 and w.stride(0) < w.shape[1]):
            w = w.contiguous()
            if w.is_cuda:                                     # torch's stream makes the copy, the context's reads it
                import torch
                torch.cuda.current_stream(w.device).synchronize()
        return w.data_ptr(), (w.stride(0) if w.shape[0] > 1 else w.shape[1]), w

    def apply_device(self, rows: AdapterRows, x, base, out) -> None:
        """out[p] = base[p] + scale * B (A x[p]) for the assigned rows (float32 device rows; out may be base)."""
        device = self.ctx.device
        xp, ldx, _ = _rows(x, rows.rows, self.columns, "x", device, (_lib.F32,))
        bp, ldb, _ = _rows(base, rows.rows, self.rows, "base", device, (_lib.F32,))
        op, ldo, _ = _rows(out, rows.rows, self.rows, "out", device, (_lib.F32,))
        check(_lib.lib().satori_adapters_apply_device(self.handle, rows.handle, xp, ldx, bp, ldb, op, ldo),
              "adapters_apply")

    def execute_device(self, matrix: CudaQuantizedMatrix, rows: AdapterRows, x, out, order: int = _lib.ORDER_BATCH) -> None:
        """The quantized projection of the assigned rows with their adapters added (packed float32 rows)."""
        device = self.ctx.device
        xp, ldx, _ = _rows(x, rows.rows, self.columns, "x", device, (_lib.F32,))
        op, ldo, _ = _rows(out, rows.rows, self.rows, "out", device, (_lib.F32,))
        if ldx != self.columns or ldo != self.rows:
            raise _bad("x and out must be packed")
        check(_lib.lib().satori_matrix_execute_adapted_device(matrix.handle, self.handle, rows.handle, xp, op, order),
              "execute_adapted")

    def dispose(self) -> None:
        if self._h:
            if _open(self.ctx):
                _lib.lib().satori_adapters_destroy(self._h)
            self._h = _vp()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass
