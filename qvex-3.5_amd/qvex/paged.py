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

import ctypes

import torch

from . import _C
from .kernels import _check

FORMATS = {"bf16": (0, torch.bfloat16), "int8": (1, torch.int8), "fp8": (2, torch.float8_e4m3fn)}
_OF_DTYPE = {t: n for n, (_, t) in FORMATS.items()}


class KVPages:
    """The tensors of a pool: k, v [n_pages, n_kv, page, head_dim] in bf16, int8 or
    float8_e4m3fn, and for the 8-bit types k_scale, v_scale fp32 [n_pages, n_kv, page]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dtype not in _OF_DTYPE:
            raise _C.QvexError(f"pages must be bf16, int8 or float8_e4m3fn (got {k.dtype})")
        self.fmt = _OF_DTYPE[k.dtype]
        _check(k, "k pages", k.dtype, 4)
        _check(v, "v pages", k.dtype, 4)
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
                _check(t, n, torch.float32, 3)
                if t.shape != k.shape[:3] or t.device != k.device:
                    raise _C.QvexError(f"{n} must be {tuple(k.shape[:3])} on {k.device}")
        if self.head_dim not in (128, 256) or self.page not in (16, 32, 64, 128, 256, 512, 1024):
            raise _C.QvexError(f"pages of {self.page} x {self.head_dim}: a power of two of 16..1024 positions, "
                               "heads of 128 or 256")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        ptr = [None if t is None else t.data_ptr() for t in (k, v, k_scale, v_scale)]
        self._c = _C.KvPages(*ptr, self.n_pages, self.page, self.n_kv, self.head_dim, FORMATS[self.fmt][0])
        self._ref = ctypes.byref(self._c)

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
        if torch.cuda.current_device() != self.device.index:
            raise _C.QvexError(f"the pages are on {self.device}, the current device is "
                               f"cuda:{torch.cuda.current_device()}")
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    def _rows(self, table, pos, T: int, cu, max_rows):
        dev = self.device
        B = pos.shape[0] if pos.dim() == 1 else -1
        if pos.dtype != torch.int32 or pos.device != dev or B < 1 or not pos.is_contiguous():
            raise _C.QvexError(f"pos must be a contiguous int32 [B] tensor on {dev} "
                               f"(got {pos.dtype} {tuple(pos.shape)} on {pos.device})")
        if table.dtype != torch.int32 or table.device != dev or table.dim() != 2 or table.shape[0] != B \
                or table.shape[1] < 1 or (table.stride(1) != 1 and table.shape[1] > 1):
            raise _C.QvexError(f"table must be int32 [B = {B}, W] on {dev} with consecutive entries "
                               f"(got {table.dtype} {tuple(table.shape)} on {table.device})")
        if cu is None:
            if T % B:
                raise _C.QvexError(f"{T} rows do not divide over {B} sequences: row offsets (cu) are needed")
            L, cp = T // B, None
        else:
            if cu.dtype != torch.int32 or cu.device != dev or cu.shape != (B + 1,) or not cu.is_contiguous():
                raise _C.QvexError(f"cu must be a contiguous int32 [B + 1 = {B + 1}] tensor on {dev} "
                                   f"(got {cu.dtype} {tuple(cu.shape)} on {cu.device})")
            L, cp = T if max_rows is None else max(1, min(int(max_rows), T)), cu.data_ptr()
        return ctypes.byref(_C.KvRows(table.data_ptr(), pos.data_ptr(), cp, table.stride(0), table.shape[1], B, L, T)), B, L

    def _heads(self, t, name: str, T: int | None, heads: int | None):
        """A bf16 [T, heads, head_dim] view with consecutive dims on this device."""
        if t.dtype != torch.bfloat16 or t.device != self.device or t.dim() != 3 or t.shape[2] != self.head_dim \
                or t.stride(2) != 1 or (T is not None and t.shape[0] != T) or (heads is not None and t.shape[1] != heads):
            raise _C.QvexError(f"{name} must be bf16 [{'T' if T is None else T}, {'H' if heads is None else heads}, "
                               f"{self.head_dim}] on {self.device} with consecutive dims (got {t.dtype} "
                               f"{tuple(t.shape)} on {t.device})")


def kv_append(pages: KVPages, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, pos: torch.Tensor,
              cu: torch.Tensor | None = None, max_rows: int | None = None) -> None:
    """Write rows k, v bf16 [T, n_kv, head_dim] (any row and head strides) at their
    sequences' next positions, quantized to the pages' format (KVCache.update,
    engine/model.py:156-170). max_rows: the most rows of a sequence, where known (speed only)."""
    T = k.shape[0]
    pages._heads(k, "k", None, pages.n_kv)
    pages._heads(v, "v", T, pages.n_kv)
    if T == 0:
        return
    rows, _, _ = pages._rows(table, pos, T, cu, max_rows)
    _C.call("qvex_paged_append", pages._ref, rows, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
            v.stride(1), pages._stream())


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
    if proj.dtype != torch.bfloat16 or proj.device != pages.device or proj.dim() != 2 or proj.stride(1) != 1:
        raise _C.QvexError(f"proj must be bf16 [T, width] on {pages.device} with consecutive columns "
                           f"(got {proj.dtype} {tuple(proj.shape)} on {proj.device})")
    T, width = proj.shape
    Hq = width // (2 * D) - pages.n_kv
    if width % (2 * D) or Hq < 1 or Hq % pages.n_kv:
        raise _C.QvexError(f"proj rows of {width} are not [Hq x (q | gate) | k | v] with {pages.n_kv} kv heads of {D}")
    for t, n in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t.dtype != torch.bfloat16 or t.device != pages.device or t.shape != (D,) or not t.is_contiguous():
            raise _C.QvexError(f"{n} must be a contiguous bf16 [{D}] tensor on {pages.device}")
    rot = 0
    if freqs is not None:
        if freqs.dtype != torch.float64 or freqs.device != pages.device or freqs.dim() != 1 or not freqs.is_contiguous():
            raise _C.QvexError(f"freqs must be a contiguous fp64 [rot / 2] tensor on {pages.device}")
        rot = 2 * freqs.numel()
    if q_out is None:
        q_out = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=proj.device)
    elif q_out.dtype != torch.bfloat16 or q_out.device != pages.device or q_out.shape != (T, Hq, D) \
            or not q_out.is_contiguous():
        raise _C.QvexError(f"q_out must be a contiguous bf16 {(T, Hq, D)} tensor on {pages.device}")
    if T == 0:
        return q_out
    rows, _, _ = pages._rows(table, pos, T, cu, max_rows)
    _C.call("qvex_paged_qk_rope", pages._ref, rows, proj.data_ptr(), proj.stride(0) if T > 1 else width,
            q_norm.data_ptr(), k_norm.data_ptr(), Hq, rot, freqs.data_ptr() if rot else None, float(eps),
            q_out.data_ptr(), pages._stream())
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
    out = []
    for t, n in ((k_out, "k_out"), (v_out, "v_out")):
        if t is None:
            t = torch.empty(shape, dtype=dtype, device=pages.device)
        elif t.dtype != dtype or t.device != pages.device or t.shape != shape or not t.is_contiguous():
            raise _C.QvexError(f"{n} must be a contiguous {dtype} {shape} tensor on {pages.device}")
        out.append(t)
    if T:
        rows, _, _ = pages._rows(table, pos, T, cu, max_rows)
        _C.call("qvex_paged_read", pages._ref, rows, out[0].data_ptr(), out[1].data_ptr(),
                int(dtype == torch.float32), pages._stream())
    return out[0], out[1]


def attention(pages: KVPages, q: torch.Tensor, table: torch.Tensor, pos: torch.Tensor, max_keys: int | None = None,
              cu: torch.Tensor | None = None, max_rows: int | None = None, gate: torch.Tensor | None = None,
              scale: float | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
              keys_per_split: int = 0) -> torch.Tensor:
    """Causal GQA attention of rows q bf16 [T, Hq, D] (any row and head strides) over
    their sequences' pages: row i of sequence b sees positions 0 .. pos[b] + i (append
    the rows' own keys first). gate [T, Hq, D]: the output times sigmoid(gate)
    (engine/model.py:228-232). scale: 1 / sqrt(D) if None. max_keys: a bound of pos[b] +
    rows, the table's capacity if None. keys_per_split: see qvex_paged_attention.
    workspace: any tensor of at least workspace_bytes(); one is made per call if None.
    Returns bf16 [T, Hq, D]; rows outside every sequence are left as they are in out."""
    T, Hq = q.shape[0], q.shape[1] if q.dim() == 3 else 0
    pages._heads(q, "q", None, None)
    if Hq < 1 or Hq % pages.n_kv:
        raise _C.QvexError(f"{Hq} query heads do not share {pages.n_kv} kv heads")
    D = pages.head_dim
    if gate is not None:
        pages._heads(gate, "gate", T, Hq)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=q.device)
    elif out.dtype != torch.bfloat16 or out.device != pages.device or out.shape != (T, Hq, D) or not out.is_contiguous():
        raise _C.QvexError(f"out must be a contiguous bf16 {(T, Hq, D)} tensor on {pages.device}")
    if T == 0:
        return out
    rows, B, L = pages._rows(table, pos, T, cu, max_rows)
    cap = table.shape[1] * pages.page
    mk = cap if max_keys is None else max(1, min(int(max_keys), cap))
    need = _C.lib().qvex_paged_attention_workspace_bytes(B, L, T, Hq, pages.n_kv, D, mk, int(keys_per_split))
    have, wp = 0, None
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif workspace.device != pages.device or not workspace.is_contiguous():
            raise _C.QvexError(f"workspace must be a contiguous tensor on {pages.device}")
        have, wp = workspace.numel() * workspace.element_size(), workspace.data_ptr()
    _C.call("qvex_paged_attention", pages._ref, rows, q.data_ptr(), q.stride(0), q.stride(1), Hq, mk,
            int(keys_per_split), None if gate is None else gate.data_ptr(), 0 if gate is None else gate.stride(0),
            0 if gate is None else gate.stride(1), D ** -0.5 if scale is None else float(scale), out.data_ptr(), wp, have,
            pages._stream())
    return out


def workspace_bytes(pages: KVPages, B: int, T: int, Hq: int, max_keys: int, max_rows: int | None = None,
                    keys_per_split: int = 0) -> int:
    """Bytes of workspace that attention() takes for T rows of B sequences (0: none)."""
    L = (T // B if T % B == 0 else T) if max_rows is None else max(1, min(int(max_rows), T))
    return int(_C.lib().qvex_paged_attention_workspace_bytes(B, L, T, Hq, pages.n_kv, pages.head_dim, int(max_keys),
                                                             int(keys_per_split)))
