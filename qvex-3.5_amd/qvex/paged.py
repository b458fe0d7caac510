"""Paged KV cache: pages of keys and values in bf16 or quantized to 8 bits as they
are written, and the attention that reads them.

``KVPages`` holds the tensors of a pool. The functions take a call's rows as a
ragged batch: ``table`` int32 [B, W] (the pages of each sequence in order, -1
for none), ``pos`` int32 [B] (positions held before the call) and ``cu`` int32
[B + 1] (row offsets of the sequences; None: T / B rows each). All three live on
the device and are checked there: a row whose position has no page is not
written, reads as zeros, and is not seen by attention. Formats: ``bf16``, ``int8``
(codes -127..127) and ``fp8`` (e4m3), the latter two with an fp32 scale per
position and kv head (include/qvex.h has the definitions).

The reference keeps one dense bf16 array per sequence (KVCache,
engine/model.py:149-176), which a longer prompt moves and a shared prefix copies.
"""

from __future__ import annotations

import functools
import weakref

import torch

from . import _C

_BF16, _I32, _F64 = torch.bfloat16, torch.int32, torch.float64
FORMATS = {"bf16": (0, torch.bfloat16), "int8": (1, torch.int8), "fp8": (2, torch.float8_e4m3fn)}
_OF_DTYPE = {t: n for n, (_, t) in FORMATS.items()}


class _Entry:
    """An entry point of the library, looked up at its first call (a decode step makes
    these calls per layer: 0.5 us less than _C.call each)."""

    def __init__(self, name: str):
        self.name, self.fn = name, None

    def __call__(self, *args) -> None:
        if self.fn is None:
            self.fn = getattr(_C.lib(), self.name)
        rc = self.fn(*args)
        if rc != 0:
            raise _C.QvexError(f"{self.name} failed (status {rc}): {_C.lib().qvex_last_error().decode(errors='replace')}")


_append, _qk_rope, _read, _attention = (_Entry("qvex_paged_" + n) for n in ("append", "qk_rope", "read", "attention"))


class KVPages:
    """The tensors of a pool: k, v [n_pages, n_kv, page, head_dim] in bf16, int8 or
    float8_e4m3fn, and for the 8-bit types k_scale, v_scale fp32 [n_pages, n_kv, page]."""

    _dev = -1       # the device's index

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dtype not in _OF_DTYPE:
            raise _C.QvexError(f"pages must be bf16, int8 or float8_e4m3fn (got {k.dtype})")
        self.fmt = _OF_DTYPE[k.dtype]
        for t, n in ((k, "k"), (v, "v")):
            if t.dtype != k.dtype or t.dim() != 4 or not t.is_contiguous():
                raise _C.QvexError(f"{n} pages must be contiguous {k.dtype} [n_pages, n_kv, page, head_dim] "
                                   f"(got {t.dtype} {tuple(t.shape)})")
        self.n_pages, self.n_kv, self.page, self.head_dim = k.shape
        if v.shape != k.shape or v.device != k.device:
            raise _C.QvexError(f"k and v pages differ: {tuple(k.shape)} on {k.device}, {tuple(v.shape)} on {v.device}")
        if self.fmt == "bf16":
            if k_scale is not None or v_scale is not None:
                raise _C.QvexError("bf16 pages have no scales")
        else:
            for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                if t is None:
                    raise _C.QvexError(f"{self.fmt} pages need {n}")
                if t.dtype != torch.float32 or t.shape != k.shape[:3] or t.device != k.device or not t.is_contiguous():
                    raise _C.QvexError(f"{n} must be contiguous fp32 {tuple(k.shape[:3])} on {k.device} (got {t.dtype} "
                                       f"{tuple(t.shape)} on {t.device})")
        if self.head_dim not in (128, 256) or self.page not in (16, 32, 64, 128, 256, 512, 1024):
            raise _C.QvexError(f"pages of {self.page} x {self.head_dim}: a power of two of 16..1024 positions, "
                               "heads of 128 or 256")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self._dev = k.device, k.get_device()
        ptr = [None if t is None else t.data_ptr() for t in (k, v, k_scale, v_scale)]
        self._c = _C.KvPages(*ptr, self.n_pages, self.page, self.n_kv, self.head_dim, FORMATS[self.fmt][0])

    @classmethod
    def alloc(cls, n_pages: int, n_kv: int, head_dim: int, fmt: str = "int8", page: int = 64, device=None) -> "KVPages":
        """A zeroed pool."""
        if fmt not in FORMATS:
            raise _C.QvexError(f"unknown KV format {fmt!r} ({', '.join(FORMATS)})")
        shape = (n_pages, n_kv, page, head_dim)
        k, v = (torch.zeros(shape, dtype=FORMATS[fmt][1], device=device) for _ in range(2))
        if fmt == "bf16":
            return cls(k, v)
        return cls(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    def tensors(self) -> list[torch.Tensor]:
        return [t for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None]

    def _stream(self) -> int:
        if self._dev < 0:
            raise _C.QvexError(f"the pages must be on a GPU (they are on {self.device})")
        if torch._C._cuda_getDevice() != self._dev:
            raise _C.QvexError(f"the pages are on {self.device}, the current device is "
                               f"cuda:{torch.cuda.current_device()}")
        return torch._C._cuda_getCurrentRawStream(self._dev)

    def _rows(self, table, pos, T: int, cu, max_rows):
        """(qvex_kv_rows, B, L, positions that a table row holds) of a call's rows."""
        dev = self._dev
        if pos.dtype is not _I32 or pos.get_device() != dev or pos.ndim != 1 or not pos.is_contiguous():
            raise _C.QvexError(f"pos must be a contiguous int32 [B] tensor on {self.device} "
                               f"(got {pos.dtype} {tuple(pos.shape)} on {pos.device})")
        B = len(pos)
        if table.dtype is not _I32 or table.get_device() != dev or table.ndim != 2:
            raise _C.QvexError(f"table must be int32 [B, W] on {self.device} (got {table.dtype} {tuple(table.shape)} "
                               f"on {table.device})")
        n, width = table.shape
        step, one = table.stride()
        if n != B or B < 1 or width < 1 or (one != 1 and width > 1):
            raise _C.QvexError(f"table must be [B = {B}, W] with consecutive entries (got {tuple(table.shape)})")
        if cu is None:
            if T % B:
                raise _C.QvexError(f"{T} rows do not divide over {B} sequences: row offsets (cu) are needed")
            L, cp = T // B, None
        else:
            if cu.dtype is not _I32 or cu.get_device() != dev or cu.shape != (B + 1,) or not cu.is_contiguous():
                raise _C.QvexError(f"cu must be a contiguous int32 [B + 1 = {B + 1}] tensor on {self.device} "
                                   f"(got {cu.dtype} {tuple(cu.shape)} on {cu.device})")
            L, cp = T if max_rows is None else max(1, min(int(max_rows), T)), cu.data_ptr()
        return (_C.KvRows(table.data_ptr(), pos.data_ptr(), cp, step, width, B, L, T), B, L, width * self.page)

    def _heads(self, t, name: str, T: int | None = None, heads: int | None = None):
        """(rows, heads, row stride, head stride) of a bf16 [T, heads, head_dim] view with consecutive dims."""
        if t.dtype is _BF16 and t.get_device() == self._dev and t.ndim == 3:
            n, h, d = t.shape
            st, sh, one = t.stride()
            if d == self.head_dim and one == 1 and (T is None or n == T) and (heads is None or h == heads):
                return n, h, st, sh
        raise _C.QvexError(f"{name} must be bf16 [{'T' if T is None else T}, {'H' if heads is None else heads}, "
                           f"{self.head_dim}] on {self.device} with consecutive dims (got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device})")

    def _out(self, t, name: str, shape, dtype):
        if t.dtype is not dtype or t.get_device() != self._dev or t.shape != shape or not t.is_contiguous():
            raise _C.QvexError(f"{name} must be a contiguous {dtype} {shape} tensor on {self.device} (got {t.dtype} "
                               f"{tuple(t.shape)} on {t.device})")


def kv_append(pages: KVPages, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, pos: torch.Tensor,
              cu: torch.Tensor | None = None, max_rows: int | None = None) -> None:
    """Write rows k, v bf16 [T, n_kv, head_dim] (any row and head strides) at their
    sequences' next positions, quantized to the pages' format (KVCache.update,
    engine/model.py:156-170). max_rows: the most rows of a sequence, where known (speed only)."""
    T, _, kt, kh = pages._heads(k, "k", None, pages.n_kv)
    _, _, vt, vh = pages._heads(v, "v", T, pages.n_kv)
    if T:
        rows = pages._rows(table, pos, T, cu, max_rows)[0]
        _append(pages._c, rows, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, pages._stream())


def rope_freqs(rot: int, theta: float, device) -> torch.Tensor:
    """theta^(-2i / rot) for i < rot / 2 in fp64, for attn_qk_rope."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    return float(theta) ** (-2.0 * i / max(rot, 1))


def attn_qk_rope(pages: KVPages, proj: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, table: torch.Tensor,
                 pos: torch.Tensor, freqs: torch.Tensor | None, eps: float, cu: torch.Tensor | None = None,
                 max_rows: int | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention's input stage over pages (engine/model.py:213-226): proj bf16
    [T, Hq*2D + 2*n_kv*D] rows [Hq x (q | gate) | k | v]; q and k normalised and their first
    2 * len(freqs) dims rotated by position * freqs (rope_freqs), k and v appended as kv_append
    does. Returns q bf16 [T, Hq, D]."""
    D = pages.head_dim
    if proj.dtype is not _BF16 or proj.get_device() != pages._dev or proj.ndim != 2 or proj.stride(1) != 1:
        raise _C.QvexError(f"proj must be bf16 [T, width] on {pages.device} with consecutive columns "
                           f"(got {proj.dtype} {tuple(proj.shape)} on {proj.device})")
    T, width = proj.shape
    Hq = width // (2 * D) - pages.n_kv
    if width % (2 * D) or Hq < 1 or Hq % pages.n_kv:
        raise _C.QvexError(f"proj rows of {width} are not [Hq x (q | gate) | k | v] with {pages.n_kv} kv heads of {D}")
    for t, n in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t.dtype is not _BF16 or t.get_device() != pages._dev or t.shape != (D,) or not t.is_contiguous():
            raise _C.QvexError(f"{n} must be a contiguous bf16 [{D}] tensor on {pages.device}")
    rot = 0
    if freqs is not None:
        if freqs.dtype is not _F64 or freqs.get_device() != pages._dev or freqs.ndim != 1 or not freqs.is_contiguous():
            raise _C.QvexError(f"freqs must be a contiguous fp64 [rot / 2] tensor on {pages.device}")
        rot = 2 * len(freqs)
    if q_out is None:
        q_out = proj.new_empty((T, Hq, D))
    else:
        pages._out(q_out, "q_out", (T, Hq, D), _BF16)
    if T:
        rows = pages._rows(table, pos, T, cu, max_rows)[0]
        _qk_rope(pages._c, rows, proj.data_ptr(), proj.stride(0) if T > 1 else width, q_norm.data_ptr(),
                 k_norm.data_ptr(), Hq, rot, freqs.data_ptr() if rot else None, eps, q_out.data_ptr(), pages._stream())
    return q_out


def kv_read(pages: KVPages, table: torch.Tensor, pos: torch.Tensor, T: int, cu: torch.Tensor | None = None,
            max_rows: int | None = None, dtype: torch.dtype = torch.bfloat16, k_out: torch.Tensor | None = None,
            v_out: torch.Tensor | None = None):
    """The T rows at pos[b], pos[b] + 1, ... of each sequence read back: (k, v), each
    [T, n_kv, head_dim] in bf16 or fp32 (what kv_append with the same arguments
    wrote). Rows outside every sequence are left as they are in k_out, v_out."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise _C.QvexError(f"kv_read gives bf16 or fp32 (got {dtype})")
    T = int(T)
    shape = (T, pages.n_kv, pages.head_dim)
    if T < 0:
        raise _C.QvexError(f"kv_read: T={T}")
    if k_out is None:
        k_out = torch.empty(shape, dtype=dtype, device=pages.device)
    else:
        pages._out(k_out, "k_out", shape, dtype)
    if v_out is None:
        v_out = torch.empty_like(k_out)
    else:
        pages._out(v_out, "v_out", shape, dtype)
    if T:
        rows = pages._rows(table, pos, T, cu, max_rows)[0]
        _read(pages._c, rows, k_out.data_ptr(), v_out.data_ptr(), int(dtype is torch.float32), pages._stream())
    return k_out, v_out


def attention(pages: KVPages, q: torch.Tensor, table: torch.Tensor, pos: torch.Tensor, max_keys: int | None = None,
              cu: torch.Tensor | None = None, max_rows: int | None = None, gate: torch.Tensor | None = None,
              scale: float | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
              keys_per_split: int = 0) -> torch.Tensor:
    """Causal GQA attention of rows q bf16 [T, Hq, D] (any row and head strides) over
    their sequences' pages: row i of sequence b sees positions 0 .. pos[b] + i (append
    the rows' own keys first). gate [T, Hq, D]: the output times sigmoid(gate)
    (engine/model.py:228-232). scale: 1 / sqrt(D) if None. max_keys: a bound of pos[b] +
    rows, the table's capacity if None. keys_per_split: see qvex_paged_attention; the
    promise on a row's bits takes max_rows of 8 or less where cu is given.
    workspace: any tensor of at least workspace_bytes(); one is made per call if None.
    Returns bf16 [T, Hq, D]; rows outside every sequence are left as they are in out."""
    T, Hq, qt, qh = pages._heads(q, "q")
    if Hq < 1 or Hq % pages.n_kv:
        raise _C.QvexError(f"{Hq} query heads do not share {pages.n_kv} kv heads")
    D = pages.head_dim
    gp, gt, gh = None, 0, 0
    if gate is not None:
        _, _, gt, gh = pages._heads(gate, "gate", T, Hq)
        gp = gate.data_ptr()
    if out is None:
        out = q.new_empty((T, Hq, D))
    else:
        pages._out(out, "out", (T, Hq, D), _BF16)
    if T == 0:
        return out
    rows, B, L, cap = pages._rows(table, pos, T, cu, max_rows)
    mk = cap if max_keys is None else max(1, min(int(max_keys), cap))
    need = _workspace_bytes(B, L, T, Hq, pages.n_kv, D, mk, keys_per_split)
    have, wp = 0, None
    if need:
        if workspace is None:
            workspace = q.new_empty((need + 1) // 2)
        elif workspace.get_device() != pages._dev or not workspace.is_contiguous():
            raise _C.QvexError(f"workspace must be a contiguous tensor on {pages.device}")
        have, wp = workspace.nbytes, workspace.data_ptr()
    _attention(pages._c, rows, q.data_ptr(), qt, qh, Hq, mk, keys_per_split, gp, gt, gh,
               D ** -0.5 if scale is None else scale, out.data_ptr(), wp, have, pages._stream())
    return out


@functools.lru_cache(maxsize=256)
def _workspace_bytes(*args) -> int:
    return _C.lib().qvex_paged_attention_workspace_bytes(*args)


def workspace_bytes(pages: KVPages, B: int, T: int, Hq: int, max_keys: int, max_rows: int | None = None,
                    keys_per_split: int = 0) -> int:
    """Bytes of workspace that attention() takes for T rows of B sequences (0: none), with cu or
    without, at this max_keys or any smaller one. max_keys as there, at most the table's capacity."""
    widths = {T if max_rows is None else max(1, min(int(max_rows), T)), T // B}
    return max(_workspace_bytes(B, L, T, Hq, pages.n_kv, pages.head_dim, int(max_keys), int(keys_per_split))
               for L in widths)


# ---------------------------------------------------------------- pages handed to sequences

class PagePool:
    """A pool's pages and who holds them: ``take`` gives free pages, ``share`` adds a
    holder (a prefix that two sequences have in common), ``give`` ends a hold. A page
    with several holders is only read. growable: ``take`` enlarges the pool when
    it runs out, as KVCache.grow does (the tensors move; refused while a captured
    cycle drives a cache of the pool); otherwise running out raises.

    Pages change hands in the order of the calls: caches of one pool are used on one
    stream, or the caller orders their streams."""

    def __init__(self, n_pages: int, n_kv: int, head_dim: int, fmt: str = "int8", page: int = 64, device=None,
                 growable: bool = False):
        self.pages = KVPages.alloc(n_pages, n_kv, head_dim, fmt, page, device)
        self.growable = growable
        self.holders = [0] * n_pages
        self.free = list(range(n_pages - 1, -1, -1))
        self.users: weakref.WeakSet = weakref.WeakSet()

    @property
    def page(self) -> int:
        return self.pages.page

    def take(self, n: int) -> list[int]:
        if n > len(self.free):
            if not self.growable:
                raise _C.QvexError(f"the page pool has {len(self.free)} free pages of {self.pages.n_pages}, {n} are needed")
            self.grow(max(n - len(self.free), self.pages.n_pages // 2))
        got = [self.free.pop() for _ in range(n)]
        for j in got:
            self.holders[j] = 1
        return got

    def share(self, ids) -> None:
        for j in ids:
            self.holders[j] += 1

    def give(self, ids) -> None:
        for j in ids:
            self.holders[j] -= 1
            if self.holders[j] == 0:
                self.free.append(j)

    def copy(self, src: int, dst: int) -> None:
        for t in self.pages.tensors():
            t[dst].copy_(t[src])

    def grow(self, n: int) -> None:
        """n more pages: larger tensors that start with the old ones' pages."""
        if any(c.counters.graph_mode for c in self.users):
            raise _C.QvexError("a captured cycle drives a cache of this page pool; release() it before the pool grows")
        old = self.pages
        new = KVPages.alloc(old.n_pages + n, old.n_kv, old.head_dim, old.fmt, old.page, old.device)
        for a, b in zip(new.tensors(), old.tensors()):
            a[:old.n_pages].copy_(b)
        self.pages = new
        self.holders += [0] * n
        self.free = list(range(new.n_pages - 1, old.n_pages - 1, -1)) + self.free


class PagedKVCache:
    """One sequence's keys and values of one layer in a pool's pages, with KVCache's
    interface (offset, rollback, grow, clone, keys, values; engine/model.py:149-176).
    Growing adds free pages of the pool to its table and moves no key (a growable pool
    that has none left moves as a whole); a clone shares the whole pages of the prefix and
    copies the one that the next key goes to. What finds too few pages raises, with
    nothing changed.

    The page of position ``offset`` and all behind it have this cache as their only holder
    (clone and rollback see to it), so an append never writes a shared page."""

    step = 256

    def __init__(self, pool: PagePool, counters=None, index: int = 0, *, capacity: int = 0):
        if counters is None:
            from .model import CacheCounters
            counters, index = CacheCounters(1, pool.pages.device), 0
        self.pool, self.counters, self.index = pool, counters, index
        self.ids: list[int] = []
        self.table = torch.full((1, 1), -1, dtype=torch.int32, device=pool.pages.device)
        self.pos = counters.dev[index:index + 1]
        pool.users.add(self)
        self._extend(max(capacity, 1))

    def __del__(self):
        if getattr(self, "ids", None):
            self.pool.give(self.ids)

    @property
    def pages(self) -> KVPages:
        return self.pool.pages

    @property
    def capacity(self) -> int:
        return len(self.ids) * self.pool.page

    @property
    def offset(self) -> int:
        return self.counters.get(self.index)

    @offset.setter
    def offset(self, v: int) -> None:
        if v < self.offset:
            self.counters._check_host_edit()
            self._own(max(v, 0))
        self.counters.set(self.index, v)

    def rollback(self, n=1):
        self.offset -= n     # entries past offset are overwritten by the next append

    def state(self):
        return self.pages.tensors()

    def _pages_for(self, min_capacity: int) -> int:
        size = -(-min_capacity // self.step) * self.step
        return -(-size // self.pool.page) - len(self.ids)

    def _extend(self, min_capacity: int) -> None:
        self.ids += self.pool.take(self._pages_for(min_capacity))
        self._upload()

    def _upload(self) -> None:
        if self.table.shape[1] < len(self.ids):
            self.table = torch.full((1, len(self.ids)), -1, dtype=torch.int32, device=self.table.device)
        self.table[0, :len(self.ids)].copy_(torch.tensor(self.ids, dtype=torch.int32))

    def _own(self, at: int) -> None:
        """The pages from position `at` on become this cache's alone (those behind `offset` are).
        All of them are taken first: a pool that cannot give them raises with nothing changed."""
        page, holders = self.pool.page, self.pool.holders
        first = at // page
        shared = [x for x in range(first, min(self.offset // page + 1, len(self.ids))) if holders[self.ids[x]] > 1]
        if not shared:
            return
        fresh, old = self.pool.take(len(shared)), [self.ids[x] for x in shared]
        if shared[0] == first and at % page:
            self.pool.copy(old[0], fresh[0])
        for x, j in zip(shared, fresh):
            self.ids[x] = j
        self._upload()
        self.pool.give(old)

    def grow(self, min_capacity: int) -> bool:
        """Pages for at least min_capacity positions, in steps of 256 (a HIP graph
        captured on the cache must be captured again). Returns whether any were added."""
        self.counters._check_host_edit()
        if min_capacity <= self.capacity:
            return False
        self._extend(min_capacity)
        return True

    @staticmethod
    def grow_all(caches, extra: int) -> bool:
        """Pages for `extra` positions past the offset of every paged cache among `caches`, or, where a
        pool cannot give them, an error with none of them changed. Returns whether any grew."""
        short = [c for c in caches if isinstance(c, PagedKVCache) and c.offset + extra > c.capacity]
        for c in short:
            c.counters._check_host_edit()
        got = []
        try:
            for c in short:
                got.append((c, c.pool.take(c._pages_for(c.offset + extra))))
        except BaseException:
            for c, ids in got:
                c.pool.give(ids)
            raise
        for c, ids in got:
            c.ids += ids
            c._upload()
        return bool(got)

    def clone(self, counters=None) -> "PagedKVCache":
        """A cache of the same keys that shares the prefix's whole pages; counters:
        the cloned table it indexes (a new one-entry table for a standalone cache).
        Its capacity is what the prefix needs, and grows."""
        c = PagedKVCache.__new__(PagedKVCache)
        c.pool = self.pool
        c.counters = counters if counters is not None else self.counters.clone()
        c.index, c.ids = self.index, []
        c.pos = c.counters.dev[c.index:c.index + 1]
        n = self.offset // self.pool.page
        size = -(-(self.offset + 1) // self.step) * self.step
        c.ids = fresh = self.pool.take(-(-size // self.pool.page) - n)   # given back if what follows raises
        if self.offset % self.pool.page:
            self.pool.copy(self.ids[n], fresh[0])
        self.pool.share(self.ids[:n])
        c.ids = self.ids[:n] + fresh
        c.table = torch.full((1, len(c.ids)), -1, dtype=torch.int32, device=self.table.device)
        c._upload()
        self.pool.users.add(c)
        return c

    def _rows(self) -> torch.Tensor:
        return torch.zeros(1, dtype=torch.int32, device=self.table.device)

    def keys(self) -> torch.Tensor:
        """K as bf16 [n_kv, capacity, D] (a copy)."""
        return kv_read(self.pages, self.table, self._rows(), self.capacity)[0].transpose(0, 1).contiguous()

    def values(self) -> torch.Tensor:
        """V as bf16 [n_kv, capacity, D] (a copy)."""
        return kv_read(self.pages, self.table, self._rows(), self.capacity)[1].transpose(0, 1).contiguous()
