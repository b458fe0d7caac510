"""The paged KV cache's operators as cases that can be timed and checked.

A pool of pages holds keys and values of ``page`` positions of every kv head, in
bf16 or, with a scale per position and head, in 8 bits (``int8``, or ``fp8``:
e4m3). A sequence names its pages in a row of a block table; ``pos`` counts the
positions that it holds, ``cu`` the rows of each sequence in a call's tensors.
Kinds:

``append``  new keys and values, quantized as they are written
``input``   the attention block's input stage on projection rows: q and k norms,
            rotation, and the append
``read``    a range of positions read back as bf16
``attend``  new tokens' gated attention over the pages, causal among themselves

Sizes are those of ``qvex.model.Config`` (16 query and 4 kv heads of 256, the tiny
4 and 2 of 128), its 512-token prompt chunks, verify calls of up to 8 rows and
8192-token contexts, and batches of sequences that a server runs together.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TOP = {"int8": 127.0, "fp8": 448.0}      # the largest code of each 8-bit format
TINY = 1e-30                             # a row below this is a row of zeros
THETA, EPS, ROT = 1e7, 1e-6, {256: 64, 128: 32}

_9B = {"hq": 16, "hkv": 4, "d": 256}
_TINY = {"hq": 4, "hkv": 2, "d": 128}


def listed():
    return [
        # the tokens of a decode step of 64 sequences, written in 8 bits
        {"name": "append_decode_64", "kind": "append", "fmt": "int8", "batch": 64, "rows": 1, "ctx": 8192, "ragged": True,
         "page": 64, **_9B},
        # eight prompts' chunks of up to 512 tokens at once
        {"name": "append_chunks_8", "kind": "append", "fmt": "fp8", "batch": 8, "rows": 512, "ctx": 4096, "ragged": True,
         "page": 64, **_9B},
        # the attention block's input stage of a k = 3 verify call, and of a prompt chunk
        {"name": "input_verify_4", "kind": "input", "fmt": "fp8", "batch": 1, "rows": 4, "ctx": 4096, "ragged": False,
         "page": 64, **_9B},
        {"name": "input_chunk_512", "kind": "input", "fmt": "int8", "batch": 1, "rows": 512, "ctx": 3584, "ragged": False,
         "page": 64, **_9B},
        # a short prefix of the small model, and four whole contexts, read back
        {"name": "read_prefix_300", "kind": "read", "fmt": "bf16", "batch": 1, "rows": 300, "ctx": 0, "ragged": False,
         "page": 16, **_TINY},
        {"name": "read_contexts_4", "kind": "read", "fmt": "int8", "batch": 4, "rows": 8192, "ctx": 0, "ragged": False,
         "page": 64, **_9B},
        # one token after a 4096-token prompt, and a verify call of four at an odd position
        {"name": "attend_decode_1", "kind": "attend", "fmt": "int8", "batch": 1, "rows": 1, "ctx": 4096, "ragged": False,
         "page": 64, "gate": True, **_9B},
        {"name": "attend_verify_4", "kind": "attend", "fmt": "fp8", "batch": 1, "rows": 4, "ctx": 7001, "ragged": False,
         "page": 32, "gate": True, **_9B},
        # a decode step of 64 sequences at contexts of their own
        {"name": "attend_decode_64", "kind": "attend", "fmt": "int8", "batch": 64, "rows": 1, "ctx": 8192, "ragged": True,
         "page": 64, "gate": True, **_9B},
        # a prompt chunk over an unquantized cache, and one far into a long prompt
        {"name": "attend_chunk_512", "kind": "attend", "fmt": "bf16", "batch": 1, "rows": 512, "ctx": 3584, "ragged": False,
         "page": 64, "gate": True, **_9B},
        {"name": "attend_chunk_long", "kind": "attend", "fmt": "int8", "batch": 1, "rows": 512, "ctx": 16384,
         "ragged": False, "page": 64, "gate": True, **_9B},
        # prompts' chunks and decode steps of the small model in one call
        {"name": "attend_mixed_12", "kind": "attend", "fmt": "fp8", "batch": 12, "rows": 200, "ctx": 1500, "ragged": True,
         "page": 16, "gate": False, **_TINY},
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "input", "read", "attend", "attend", "attend"])
    heads = rng.choice([_9B, _9B, _TINY, {"hq": 8, "hkv": 8, "d": 128}, {"hq": 12, "hkv": 4, "d": 128},
                        {"hq": 16, "hkv": 1, "d": 256}])
    case = {"kind": kind, "fmt": rng.choice(["int8", "int8", "fp8", "fp8", "bf16"]), "ragged": rng.random() < 0.5,
            "page": rng.choice([16, 32, 64, 64, 128, 256]), **heads}
    if kind == "read":
        batch = _loguniform(rng, 1, 16)
        rows, ctx = _loguniform(rng, 1, 32768 // batch), rng.choice([0, _loguniform(rng, 1, 1000)])
    elif kind == "attend":
        case["gate"] = rng.random() < 0.5
        if rng.random() < 0.5:                                   # decode and verify calls
            batch = _loguniform(rng, 1, 64)
            rows, ctx = rng.choice([1, 1, 2, 4, 8]), rng.choice([0, _loguniform(rng, 1, 8192)])
        else:                                                    # prompt chunks
            batch = _loguniform(rng, 1, 8)
            rows, ctx = _loguniform(rng, 9, max(9, 512 // batch)), rng.choice([0, _loguniform(rng, 1, 16384 // batch)])
    else:
        batch = _loguniform(rng, 1, 64)
        rows, ctx = _loguniform(rng, 1, 2048 // batch), rng.choice([0, _loguniform(rng, 1, 8192)])
    return {**case, "batch": batch, "rows": rows, "ctx": ctx}


# ---------------------------------------------------------------- sizes and inputs

def _layout(case):
    """Rows of each sequence and the positions that it holds before them, on the host."""
    n, rows, ctx = case["batch"], case["rows"], case["ctx"]
    if not case["ragged"]:
        return [rows] * n, [ctx] * n
    r = random.Random(131 * n + 17 * rows + ctx)
    return ([rows if i == 0 else r.randint(1, rows) for i in range(n)],
            [ctx if i == 0 else r.randint(ctx // 8, ctx) for i in range(n)])


def _rows(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _key_gain(gen, case):
    """Keys have a few channels far above the others."""
    g = torch.ones(case["d"], device=DEV)
    g[torch.randperm(case["d"], generator=gen, device=DEV)[:case["d"] // 32]] = 4.0
    return g


def _stored(x, fmt):
    """Rows x [..., D] as a page holds them: codes (or bf16) and scales (or None)."""
    if fmt == "bf16":
        return x.to(BF16), None
    x = x.float()
    top = x.abs().amax(dim=-1)
    live = top >= TINY
    # a code next to a border goes by the last bit of the factor: both quotients are rounded correctly
    inv = torch.where(live, (TOP[fmt] / top.double()).float(), torch.zeros_like(top))
    scaled = x * inv[..., None]
    codes = scaled.round().to(torch.int8) if fmt == "int8" else scaled.to(torch.float8_e4m3fn)
    return codes, torch.where(live, (top.double() / TOP[fmt]).float(), torch.zeros_like(top))


def _values(codes, scales):
    return codes.float() if scales is None else codes.float() * scales[..., None]


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1_000_003 * int(seed) + 29)
    lens, pos = _layout(case)
    P, hq, hkv, d, n = case["page"], case["hq"], case["hkv"], case["d"], case["batch"]
    T = sum(lens)
    width = -(-max(p + m for p, m in zip(pos, lens)) // P)
    need = [-(-(p + m) // P) for p, m in zip(pos, lens)]
    pages = sum(need) + 8
    # the pages of a pool that has been in use lie in no order; unused entries of the table name none
    free = torch.randperm(pages, generator=gen, device=DEV, dtype=torch.int32)
    used = torch.arange(width, device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    table[used] = free[:sum(need)]
    cu = [0]
    for m in lens:
        cu.append(cu[-1] + m)
    s = {"case": case, "table": table, "pos": torch.tensor(pos, dtype=torch.int32, device=DEV),
         "cu": torch.tensor(cu, dtype=torch.int32, device=DEV) if case["ragged"] else None,
         "max_rows": max(lens), "max_keys": max(p + m for p, m in zip(pos, lens)), "rows": T,
         # of each row: its sequence and its place in it
         "row_seq": torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(lens, device=DEV)),
         "row_at": torch.cat([torch.arange(m, device=DEV) for m in lens])}
    shape = (pages, hkv, P, d)
    gain = _key_gain(gen, case)
    if case["kind"] in ("append", "input"):
        dtype = {"bf16": BF16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}[case["fmt"]]
        s["k_pages"], s["v_pages"] = (torch.zeros(shape, dtype=dtype, device=DEV) for _ in range(2))
        s["k_scales"], s["v_scales"] = (None if case["fmt"] == "bf16" else torch.zeros(shape[:3], device=DEV)
                                        for _ in range(2))
    else:
        s["k_pages"], s["k_scales"] = _stored(_rows(gen, *shape) * gain, case["fmt"])
        s["v_pages"], s["v_scales"] = _stored(_rows(gen, *shape), case["fmt"])
    if case["kind"] == "append":     # the k and v columns of a projection's rows
        kv = torch.cat([_rows(gen, T, hkv, d) * gain, _rows(gen, T, hkv, d)], dim=1).to(BF16)
        s["k"], s["v"] = kv[:, :hkv], kv[:, hkv:]
    if case["kind"] == "input":      # [q | gate] of each query head, then k, then v
        s["proj"] = _rows(gen, T, hq * 2 * d + 2 * hkv * d).to(BF16)
        s["q_norm"] = (1.0 + 0.1 * _rows(gen, d)).to(BF16)
        s["k_norm"] = ((1.0 + 0.1 * _rows(gen, d)) * gain).to(BF16)
        half = ROT[d] // 2
        s["freqs"] = THETA ** (-torch.arange(half, dtype=F64, device=DEV) / half)
    if case["kind"] == "attend":
        s["q"] = _rows(gen, T, hq, d).to(BF16)
        s["gate"] = _rows(gen, T, hq, 2 * d).to(BF16)[..., d:] if case["gate"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:                          # the handle that a program keeps of its pool
        s["pool"] = _paged().KVPages(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    return s


def _paged():
    path = os.path.join(os.getcwd(), "qvex-3.5_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from qvex import paged
    return paged


# ---------------------------------------------------------------- plain forms

def _slots(s):
    """The page and the slot of each row's position."""
    P = s["case"]["page"]
    at = s["pos"].long()[s["row_seq"]] + s["row_at"]
    return s["table"].long()[s["row_seq"], at // P], at % P


def _write(s, k, v):
    page, slot = _slots(s)
    for name, x in (("k", k), ("v", v)):
        codes, scales = _stored(x, s["case"]["fmt"])
        pages = s[name + "_pages"]
        if scales is None:
            pages[page, :, slot] = codes
        else:
            pages.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
            s[name + "_scales"][page, :, slot] = scales


def _read(s):
    page, slot = _slots(s)
    out = []
    for name in ("k", "v"):
        scales = s[name + "_scales"]
        # fp8 tensors are gathered as bytes: indexing is not defined on them
        pages = s[name + "_pages"]
        codes = pages.view(torch.uint8)[page, :, slot].view(pages.dtype) if scales is not None else pages[page, :, slot]
        out.append(_values(codes, None if scales is None else scales[page, :, slot]).to(BF16))
    return out


def _written(s, read):
    """The cache after an append: its pages and scales, or, of 8-bit whole numbers, the values that they stand for."""
    if s["case"]["fmt"] == "int8":
        k, v = read()
        return {"k": k, "v": v, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    return {"k": s["k_pages"], "v": s["v_pages"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _input(s):
    case, proj = s["case"], s["proj"].float()
    hq, hkv, d, T = case["hq"], case["hkv"], case["d"], s["rows"]
    half = ROT[d] // 2
    at = (s["pos"].long()[s["row_seq"]] + s["row_at"]).double()
    angle = at[:, None] * s["freqs"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, w):
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w.float()
        lo, hi = x[..., :half], x[..., half:2 * half]
        return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, x[..., 2 * half:]], dim=-1)

    q = rotated(proj[:, :2 * hq * d].reshape(T, hq, 2 * d)[..., :d], s["q_norm"])
    k = rotated(proj[:, 2 * hq * d:][:, :hkv * d].reshape(T, hkv, d), s["k_norm"])
    _write(s, k, proj[:, 2 * hq * d + hkv * d:].reshape(T, hkv, d))
    return q.to(BF16)


def _attend(s):
    case = s["case"]
    hq, hkv, d, P, n = case["hq"], case["hkv"], case["d"], case["page"], case["batch"]
    keys, rows = s["max_keys"], s["max_rows"]
    at = torch.arange(keys, device=DEV)
    page, slot = s["table"].long().clamp(min=0)[:, at // P], at % P

    def gathered(name):                                            # [n, hkv, keys, d]
        pages, scales = s[name + "_pages"], s[name + "_scales"]
        codes = pages.view(torch.uint8)[page, :, slot].view(pages.dtype) if scales is not None else pages[page, :, slot]
        return _values(codes, None if scales is None else scales[page, :, slot]).transpose(1, 2)

    q = torch.zeros((n, rows, hq, d), device=DEV)
    q[s["row_seq"], s["row_at"]] = s["q"].float()
    q = q.reshape(n, rows, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    score = (q @ gathered("k").transpose(2, 3)) / math.sqrt(d)
    last = s["pos"].long()[:, None] + torch.arange(rows, device=DEV)
    seen = at[None, None, :] <= last[:, :, None]                   # [n, rows, keys]
    score = score.reshape(n, hkv, hq // hkv, rows, keys).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True))
    p = (p / p.sum(dim=-1, keepdim=True)).reshape(n, hkv, -1, keys)
    v = gathered("v").masked_fill((at[None, :] > last[:, -1:])[:, None, :, None], 0.0)
    o = (p @ v).reshape(n, hkv, hq // hkv, rows, d).permute(0, 3, 1, 2, 4).reshape(n, rows, hq, d)
    o = o[s["row_seq"], s["row_at"]]
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return o.to(BF16)


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        paged = _paged()
        at = {"cu": s["cu"], "max_rows": s["max_rows"]}
        if kind == "append":
            paged.kv_append(s["pool"], s["k"], s["v"], s["table"], s["pos"], **at)
        elif kind == "input":
            q = paged.attn_qk_rope(s["pool"], s["proj"], s["q_norm"], s["k_norm"], s["table"], s["pos"], s["freqs"], EPS,
                                   **at)
        elif kind == "read":
            return paged.kv_read(s["pool"], s["table"], s["pos"], s["rows"], **at)
        else:
            return paged.attention(s["pool"], s["q"], s["table"], s["pos"], s["max_keys"], gate=s["gate"], **at)
        out = _written(s, lambda: paged.kv_read(s["pool"], s["table"], s["pos"], s["rows"], **at))
    elif kind == "append":
        _write(s, s["k"], s["v"])
        out = _written(s, lambda: _read(s))
    elif kind == "input":
        q = _input(s)
        out = _written(s, lambda: _read(s))
    elif kind == "read":
        return _read(s)
    else:
        return _attend(s)
    return {"q": q, **out} if kind == "input" else out


def work(case):
    lens, pos = _layout(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    T = sum(lens)
    row = 2 * hkv * (2 * d if case["fmt"] == "bf16" else d + 4)      # a position's K and V as stored
    new = T * row
    if case["kind"] == "append":
        return {"bytes": new + T * 4 * hkv * d, "flops": 0}
    if case["kind"] == "input":
        return {"bytes": new + T * 2 * (hq + 2 * hkv) * d + T * 2 * hq * d, "flops": 0}
    if case["kind"] == "read":
        return {"bytes": new + T * 4 * hkv * d, "flops": 0}
    held = sum(p + m for p, m in zip(pos, lens)) * row
    seen = sum(m * p + m * (m + 1) // 2 for p, m in zip(pos, lens))  # (query, key) pairs
    return {"bytes": held + T * 2 * hq * d * (3 if case["gate"] else 2), "flops": 4 * hq * d * seen}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits

def _quantized64(x, fmt):
    """Rows in float64 -> (codes as values, scales) of the format; bf16 rows have no scales."""
    if fmt == "bf16":
        return x, None
    top = x.abs().amax(dim=-1, keepdim=True)
    scale = torch.where(top < TINY, 0.0, top / TOP[fmt])
    y = torch.where(scale > 0, x / scale, 0.0)
    y = y.round() if fmt == "int8" else y.float().to(torch.float8_e4m3fn).double()
    return y, scale[..., 0]


def exact(case, seed):
    s = _inputs(case, seed)
    lens, pos = _layout(case)
    P, hq, hkv, d, fmt = case["page"], case["hq"], case["hkv"], case["d"], case["fmt"]
    table = s["table"].tolist()
    start = 0
    outs = []
    pages = {n: s[n + "_pages"].double() for n in "kv"} if case["kind"] in ("append", "input") and fmt != "int8" else {}

    def held(name, b, lo, hi):
        """Positions lo .. hi - 1 of sequence b, [hi - lo, hkv, d]."""
        got = []
        for j in range(lo // P, (hi - 1) // P + 1):
            codes = s[name + "_pages"][table[b][j]].double()
            scales = s[name + "_scales"]
            got.append(codes if scales is None else codes * scales[table[b][j]].double()[..., None])
        return torch.cat(got, dim=1)[:, lo % P:][:, :hi - lo].transpose(0, 1)

    for b, (m, p) in enumerate(zip(lens, pos)):
        r = slice(start, start + m)
        start += m
        if case["kind"] == "read":
            outs.append([held("k", b, p, p + m), held("v", b, p, p + m)])
            continue
        if case["kind"] == "attend":
            k, v = held("k", b, 0, p + m), held("v", b, 0, p + m)
            i = torch.arange(p + m, device=DEV)[None, :] > p + torch.arange(m, device=DEV)[:, None]
            o = []
            for h in range(hq):
                g = h * hkv // hq
                a = (s["q"][r, h].double() @ k[:, g].T * d ** -0.5).masked_fill(i, -math.inf)
                o.append(torch.softmax(a, dim=1) @ v[:, g])
            o = torch.stack(o, dim=1)
            if case["gate"]:
                o = o / (1.0 + torch.exp(-s["gate"][r].double()))
            outs.append([o])
            continue
        q = []
        if case["kind"] == "append":
            k, v = s["k"][r].double(), s["v"][r].double()
        else:
            x = s["proj"][r].double()
            half = ROT[d] // 2
            turn = torch.polar(torch.ones((), dtype=F64, device=DEV),
                               (p + torch.arange(m, device=DEV, dtype=F64))[:, None] * s["freqs"])[:, None]

            def rotated(y, w):
                y = y / torch.sqrt((y * y).sum(dim=-1, keepdim=True) / d + EPS) * w.double()
                z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
                return torch.cat([z.real, z.imag, y[..., 2 * half:]], dim=-1)

            q = [rotated(x[:, :2 * hq * d].view(m, hq, 2, d)[:, :, 0], s["q_norm"])]
            k = rotated(x[:, 2 * hq * d:2 * hq * d + hkv * d].view(m, hkv, d), s["k_norm"])
            v = x[:, 2 * hq * d + hkv * d:].view(m, hkv, d)
        (kc, ks), (vc, vs) = _quantized64(k, fmt), _quantized64(v, fmt)
        i = 0
        while i < m:                                                  # a page at a time
            j, at = table[b][(p + i) // P], (p + i) % P
            e = min(m, i + P - at)
            for name, c, sc in (("k", kc, ks), ("v", vc, vs)):
                if pages:
                    pages[name][j, :, at:at + e - i] = c[i:e].transpose(0, 1)
                if sc is not None:
                    s[name + "_scales"][j, :, at:at + e - i] = sc[i:e].T.float()
            i = e
        if fmt == "int8":
            outs.append(q + [kc * ks[..., None], vc * vs[..., None]])
        else:
            outs.append(q)
    outs = [torch.cat(x) for x in zip(*outs)]
    if case["kind"] == "read":
        return outs
    if case["kind"] == "attend":
        return outs[0]
    # a scale is its row's largest value over a constant: held in 32 bits, half a unit of which is all that is lost here
    got = {} if fmt == "bf16" else {n + "_scales": s[n + "_scales"].double() for n in "kv"}
    got.update({"k": outs[-2], "v": outs[-1]} if fmt == "int8" else pages)
    return {"q": outs[0], **got} if case["kind"] == "input" else got
