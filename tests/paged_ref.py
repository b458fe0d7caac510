"""The paged KV cache's operators from their definitions, on the CPU: codes and
scales in correctly rounded fp32 (as include/qvex.h defines them), everything else
in float64, a position at a time."""

import math

import torch

TOP = {"int8": 127.0, "fp8": 448.0}
DTYPE = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def stored(row: torch.Tensor, fmt: str):
    """One row of fp32 values -> (codes, scale or None)."""
    if fmt == "bf16":
        return row.to(torch.bfloat16), None
    top = row.abs().max()
    if not bool(torch.isfinite(row).all()):
        return torch.zeros(row.shape).to(DTYPE[fmt]), torch.tensor(math.nan)
    if float(top) < 1e-30:
        return torch.zeros(row.shape).to(DTYPE[fmt]), torch.tensor(0.0)
    scaled = row * (torch.tensor(TOP[fmt]) / top)
    return (scaled.round() if fmt == "int8" else scaled).to(DTYPE[fmt]), top / TOP[fmt]


class Pool:
    """A pool on the CPU, with a marker in every slot."""

    def __init__(self, n_pages, n_kv, page, D, fmt, mark=3.0):
        self.n_pages, self.n_kv, self.page, self.D, self.fmt = n_pages, n_kv, page, D, fmt
        shape = (n_pages, n_kv, page, D)
        self.k, self.v = (torch.full(shape, mark).to(DTYPE[fmt]) for _ in range(2))
        self.ks, self.vs = (None if fmt == "bf16" else torch.full(shape[:3], 0.5) for _ in range(2))

    def slot(self, table_row, p):
        """(page, slot) of position p, or None."""
        if p < 0 or p // self.page >= len(table_row):
            return None
        j = int(table_row[p // self.page])
        return (j, p % self.page) if 0 <= j < self.n_pages else None

    def put(self, at, k, v):
        """k, v fp32 [n_kv, D] into a slot."""
        j, s = at
        for pages, scales, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
            for h in range(self.n_kv):
                c, sc = stored(x[h], self.fmt)
                pages[j, h, s] = c
                if scales is not None:
                    scales[j, h, s] = sc

    def get(self, at):
        """(k, v) fp32 [n_kv, D]: the values that a slot stands for (one fp32 product)."""
        j, s = at
        k, v = self.k[j, :, s].float(), self.v[j, :, s].float()
        return (k, v) if self.ks is None else (k * self.ks[j, :, s, None], v * self.vs[j, :, s, None])

    def tensors(self):
        return [t for t in (self.k, self.v, self.ks, self.vs) if t is not None]


def sequences(pos, cu, T):
    """(b, first row, rows, pos) of each sequence."""
    if cu is None:
        n = T // len(pos)
        return [(b, b * n, n, p) for b, p in enumerate(pos)]
    out = []
    for b, p in enumerate(pos):
        lo = min(max(cu[b], 0), T)
        out.append((b, lo, min(max(cu[b + 1], lo), T) - lo, p))
    return out


def append(pool, k, v, table, pos, cu=None):
    for b, first, n, p in sequences(pos, cu, k.shape[0]):
        for i in range(n):
            at = pool.slot(table[b], p + i)
            if at is not None:
                pool.put(at, k[first + i].float(), v[first + i].float())


def read(pool, table, pos, T, cu=None, fill=0.0):
    k, v = (torch.full((T, pool.n_kv, pool.D), fill) for _ in range(2))
    for b, first, n, p in sequences(pos, cu, T):
        for i in range(n):
            at = pool.slot(table[b], p + i)
            k[first + i], v[first + i] = pool.get(at) if at is not None else (0.0, 0.0)
    return k, v


def attention(pool, q, table, pos, cu=None, gate=None, scale=None, fill=0.0, terms=2):
    """(out, tol): the rows' attention in float64 and how far a correct kernel may be from it.

    The kernel's errors, u = 2^-24: a score is a sum of D fp32 products (D u of the sum
    of magnitudes, times 3 for its scale, its conversion to base 2 and the argument's
    subtraction), which moves its weight by as much, relatively, and the sum of
    the weights too; exp2 is good to 2 u; a weight goes into the product as two bf16 terms
    (2^-16 of it; terms=1 is a looser bound, of a weight in one term, 2^-8 of it);
    sums over n weights n u. The output is rounded to bf16 (2^-8)."""
    T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), fill, dtype=torch.float64)
    tol = torch.zeros((T, Hq, D), dtype=torch.float64)
    u = 2.0 ** -24
    for b, first, n, p in sequences(pos, cu, T):
        ks, vs, at = [], [], []
        for x in range(max(0, p + n)):
            slot = pool.slot(table[b], x)
            if slot is not None:
                kk, vv = pool.get(slot)
                ks.append(kk.double())
                vs.append(vv.double())
                at.append(x)
        if at:
            K, V, at = torch.stack(ks), torch.stack(vs), torch.tensor(at)
        for i in range(n):
            t = first + i
            out[t] = 0.0
            live = at <= p + i if len(at) else torch.zeros(0, dtype=torch.bool)
            if not bool(live.any()):
                continue
            for h in range(Hq):
                g = h * pool.n_kv // Hq
                qq = q[t, h].double()
                s = (K[live, g] @ qq) * scale
                w = torch.exp(s - s.max())
                w = w / w.sum()
                o = w @ V[live, g]
                mag = (K[live, g].abs() @ qq.abs()) * abs(scale)
                delta = 3 * (D + 8) * u * float(mag.max()) + (2 + len(w)) * u
                a = (w.abs() @ V[live, g].abs()) * (2.0 ** (-16 if terms == 2 else -8) + 2 * delta)
                if gate is not None:
                    sg = torch.sigmoid(gate[t, h].double())
                    o, a = o * sg, a * sg + o.abs() * sg * 8 * u
                out[t, h] = o
                tol[t, h] = 2.0 ** -8 * (o.abs() + a) + a
    return out, tol


def qk_rope(proj, q_norm, k_norm, Hq, n_kv, D, freqs, eps, at):
    """(q, k, v) of projection rows at positions `at`, float64."""
    T, half = proj.shape[0], len(freqs)
    x = proj.double()
    ang = at.double()[:, None] * freqs.double()
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def rot(y, w):
        y = y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + eps) * w.double()
        lo, hi = y[..., :half], y[..., half:2 * half]
        return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, y[..., 2 * half:]], dim=-1)

    q = rot(x[:, :2 * Hq * D].reshape(T, Hq, 2 * D)[..., :D], q_norm)
    k = rot(x[:, 2 * Hq * D:2 * Hq * D + n_kv * D].reshape(T, n_kv, D), k_norm)
    return q, k, x[:, 2 * Hq * D + n_kv * D:].reshape(T, n_kv, D)
