"""Paged KV cache on the GPU against its definitions on the CPU: append, read-back,
the attention block's input stage, and attention, at ragged batches, pages that end
inside a block, unused and wrong table entries, masked NaNs, strides and graphs."""

import math

import pytest
import torch

import paged_ref as ref
from qvex import paged

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "int8", "fp8"]
BF16 = torch.bfloat16


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def on(dev, *ts):
    out = [None if t is None else t.to(dev) for t in ts]
    return out[0] if len(out) == 1 else out


def gpu_pool(pool, dev):
    return paged.KVPages(*on(dev, pool.k, pool.v), *(() if pool.ks is None else on(dev, pool.ks, pool.vs)))


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    if a.dtype in (torch.float8_e4m3fn,):
        return torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    return torch.equal(torch.nan_to_num(a.float(), nan=7e9), torch.nan_to_num(b.float(), nan=7e9))


def layout(lens, pos, page, seed, spare=3, extra_width=1):
    """A table of shuffled pages for sequences of pos + lens positions, -1 behind them; its pool's size."""
    need = [max(0, -(-(p + n) // page)) for p, n in zip(pos, lens)]
    perm = torch.randperm(sum(need) + spare, generator=gen(seed)).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need)) + extra_width), -1, dtype=torch.int32)
    j = 0
    for b, m in enumerate(need):
        table[b, :m] = perm[j:j + m]
        j += m
    return table, sum(need) + spare


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------- append and read

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,n_kv,page,lens,pos", [
    (256, 4, 64, [1], [0]), (256, 4, 64, [4], [4093]), (128, 2, 16, [5, 0, 33, 1], [0, 7, 30, 15]),
    (256, 1, 32, [70, 3], [0, 1000]), (128, 8, 1024, [9, 17], [1020, 3]), (256, 3, 16, [1, 1, 1, 1, 1], [0, 15, 16, 31, 32]),
])
def test_append_and_read(dev, fmt, D, n_kv, page, lens, pos):
    """Codes, scales and every untouched slot as defined, bit for bit; read-back is code * scale rounded once."""
    g = gen(1)
    T = sum(lens)
    table, n_pages = layout(lens, pos, page, 2)
    pool = ref.Pool(n_pages, n_kv, page, D, fmt)
    # k and v as columns of one projection's rows, with a few rows of other magnitudes
    kv = torch.randn((T, 2 * n_kv, D), generator=g) * torch.exp2(torch.randint(-20, 20, (T, 2 * n_kv, 1), generator=g).float())
    kv = kv.to(BF16)
    k, v = kv[:, :n_kv], kv[:, n_kv:]
    pages = gpu_pool(pool, dev)
    cu = offsets(lens)
    kvd = kv.to(dev)
    args = (i32(table.tolist(), dev), i32(pos, dev), i32(cu, dev))
    paged.kv_append(pages, kvd[:, :n_kv], kvd[:, n_kv:], *args)
    ref.append(pool, k, v, table.tolist(), pos, cu)
    for got, want in zip(pages.tensors(), pool.tensors()):
        assert same_bits(got, want)
    for dtype in (BF16, torch.float32):
        got = paged.kv_read(pages, args[0], args[1], T, args[2], dtype=dtype)
        for x, y in zip(got, ref.read(pool, table.tolist(), pos, T, cu)):
            assert torch.equal(x.cpu(), y.to(dtype))


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_rows_that_are_not_numbers(dev, fmt):
    """Zero rows, rows below the smallest scale, NaN and infinite values: in 8 bits the whole row reads back as NaN."""
    D, n_kv, page = 128, 2, 16
    x = torch.randn((6, n_kv, D), generator=gen(3)).to(BF16)
    x[0] = 0.0
    x[1] = 1e-35
    x[2, 0, 5] = math.nan
    x[3, 1, 7] = -math.inf
    x[4, 0, 0] = torch.finfo(BF16).max
    pool = ref.Pool(2, n_kv, page, D, fmt)
    pages = gpu_pool(pool, dev)
    table, pos = i32([[1, 0]], dev), i32([3], dev)
    paged.kv_append(pages, x.to(dev), x.flip(0).contiguous().to(dev), table, pos)
    ref.append(pool, x, x.flip(0), [[1, 0]], [3])
    for got, want in zip(pages.tensors(), pool.tensors()):
        assert same_bits(got, want)
    k, _ = paged.kv_read(pages, table, pos, 6)
    if fmt != "bf16":
        assert bool(k[2, 0].isnan().all()) and not bool(k[2, 1].isnan().any()) and bool(k[3, 1].isnan().all())
    assert bool((k[0] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_and_read_where_no_page_is(dev, fmt):
    """Negative positions, positions past the table, entries outside the pool and padded rows: nothing
    is written there, zeros are read, and rows outside every sequence stay as they are."""
    D, n_kv, page = 256, 2, 16
    table = [[2, 99], [-7, 0], [1, 3]]
    pos, cu, T = [8, 10, -3], [0, 12, 20, 28], 31
    x = torch.randn((T, n_kv, D), generator=gen(4)).to(BF16)
    pool = ref.Pool(4, n_kv, page, D, fmt)
    pages = gpu_pool(pool, dev)
    args = (i32(table, dev), i32(pos, dev))
    paged.kv_append(pages, x.to(dev), (-x).to(dev), *args, i32(cu, dev), max_rows=12)
    ref.append(pool, x, -x, table, pos, cu)
    for got, want in zip(pages.tensors(), pool.tensors()):
        assert same_bits(got, want)
    k, v = (torch.full((T, n_kv, D), 5.0, dtype=BF16, device=dev) for _ in range(2))
    paged.kv_read(pages, *args, T, i32(cu, dev), k_out=k, v_out=v)
    wk, wv = ref.read(pool, table, pos, T, cu, fill=5.0)
    assert torch.equal(k.cpu(), wk.to(BF16)) and torch.equal(v.cpu(), wv.to(BF16))


def test_append_strides_and_row_bound(dev):
    """Rows and heads of any stride (odd ones too), and a row bound below the longest sequence."""
    D, n_kv, page, T = 128, 2, 32, 50
    flat = torch.randn(T * 300 + 7, generator=gen(5)).to(BF16).to(dev)
    k = flat[3:].as_strided((T, n_kv, D), (277, 133, 1))
    v = flat[1:].as_strided((T, n_kv, D), (261, 129, 1))
    pool = ref.Pool(3, n_kv, page, D, "int8")
    pages = gpu_pool(pool, dev)
    table = [[2, 0], [1, -1]]
    paged.kv_append(pages, k, v, i32(table, dev), i32([0, 0], dev), i32([0, 45, 50], dev), max_rows=1)
    ref.append(pool, k.cpu(), v.cpu(), table, [0, 0], [0, 45, 50])
    for got, want in zip(pages.tensors(), pool.tensors()):
        assert same_bits(got, want)


# ---------------------------------------------------------------- input stage

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv,rot,lens,pos,pad", [
    (256, 16, 4, 64, [4], [4096], 0), (128, 4, 2, 32, [3, 20, 1], [0, 100, 1000000], 1), (128, 2, 2, 0, [2], [5], 0),
    (128, 3, 1, 20, [7], [31], 0), (256, 8, 2, 256, [5], [77], 8),
])
def test_qk_rope(dev, fmt, D, Hq, n_kv, rot, lens, pos, pad):
    """q, and what the pages then stand for, against float64: q and bf16 rows one rounding
    (2^-8), int8 half a scale, fp8 2^-4 or half its smallest step; the fp32 chain
    (sum of squares, rsqrt, rotation of an angle reduced in fp64) adds 2^-19 of the row's largest."""
    g = gen(6)
    T, width = sum(lens), Hq * 2 * D + 2 * n_kv * D
    proj = torch.randn((T, width + pad), generator=g).to(BF16)[:, :width]
    qn, kn = (1.0 + 0.2 * torch.randn(D, generator=g)).to(BF16), (1.0 + 0.2 * torch.randn(D, generator=g)).to(BF16)
    page = 16
    tab = torch.full((len(lens), max(p + n for p, n in zip(pos, lens)) // page + 1), -1, dtype=torch.int32)
    j = 0
    for b, (p, n) in enumerate(zip(pos, lens)):
        for x in range(p // page, (p + n - 1) // page + 1):
            tab[b, x] = j
            j += 1
    pages = gpu_pool(ref.Pool(j, n_kv, page, D, fmt), dev)
    freqs = paged.rope_freqs(rot, 1e7, dev) if rot else None
    cu = offsets(lens)
    pd = torch.zeros((T, width + pad), dtype=BF16, device=dev)
    pd[:, :width] = proj.to(dev)
    args = (tab.to(dev), i32(pos, dev))
    q = paged.attn_qk_rope(pages, pd[:, :width], qn.to(dev), kn.to(dev), *args, freqs, 1e-6, i32(cu, dev))
    at = torch.cat([p + torch.arange(n) for p, n in zip(pos, lens)])
    fr = freqs.cpu() if rot else torch.zeros(0, dtype=torch.float64)
    wq, wk, wv = ref.qk_rope(proj, qn, kn, Hq, n_kv, D, fr, 1e-6, at)

    def near(got, want, rounding, floor=0.0):
        far = (got.cpu().double() - want).abs()
        assert bool((far <= rounding * want.abs() + floor + 2.0 ** -19 * want.abs().amax(dim=-1, keepdim=True)).all())

    near(q, wq, 2.0 ** -8)
    k, v = paged.kv_read(pages, *args, T, i32(cu, dev), dtype=torch.float32)
    for got, want in ((k, wk), (v, wv)):
        top = want.abs().amax(dim=-1, keepdim=True)
        if fmt == "bf16":
            near(got, want, 2.0 ** -8)
        elif fmt == "int8":
            near(got, want, 0.0, top / 254)
        else:
            near(got, want, 2.0 ** -4, top / 448 * 2.0 ** -10)


def test_qk_rope_values_are_appended_as_append_does(dev):
    """v goes to the pages with the bits of kv_append."""
    D, Hq, n_kv, T, page = 256, 4, 2, 9, 16
    proj = torch.randn((T, Hq * 2 * D + 2 * n_kv * D), generator=gen(7)).to(BF16).to(dev)
    w = torch.ones(D, dtype=BF16, device=dev)
    a, b = (paged.KVPages.alloc(2, n_kv, D, "int8", page, dev) for _ in range(2))
    table, pos = i32([[1, 0]], dev), i32([11], dev)
    paged.attn_qk_rope(a, proj, w, w, table, pos, paged.rope_freqs(64, 1e7, dev), 1e-6)
    v = proj[:, -n_kv * D:].view(T, n_kv, D)
    paged.kv_append(b, v, v, table, pos)
    assert torch.equal(a.v, b.v) and torch.equal(a.v_scale, b.v_scale)


# ---------------------------------------------------------------- attention

def check_attention(dev, fmt, D, Hq, n_kv, page, lens, pos, *, gate=False, scale=None, seed=8, poison=True, kps=0,
                    max_keys=None, max_rows=None, pad=0, fill_gain=1.0, edit=None, wide=False):
    """wide: a table of many unused entries, whose capacity as the bound of the keys makes a call of many
    rows a large one, so that it takes the form of prompt chunks."""
    g = gen(seed)
    T = sum(lens) + pad
    extra = -(-1_300_000_000 // (T * Hq * D * page)) if wide else 1
    table, n_pages = layout(lens, pos, page, seed + 1, extra_width=extra)
    pool = ref.Pool(n_pages, n_kv, page, D, fmt)
    if poison:          # what no sequence holds is no data
        if fmt == "bf16":
            pool.k[:], pool.v[:] = math.nan, math.inf
        else:
            pool.ks[:], pool.vs[:] = math.nan, math.inf
            if fmt == "fp8":
                pool.k[:], pool.v[:] = math.nan, math.nan
    for b, (p, n) in enumerate(zip(pos, lens)):
        for x in range(max(0, p + n)):
            at = pool.slot(table[b].tolist(), x)
            pool.put(at, fill_gain * torch.randn((n_kv, D), generator=g), torch.randn((n_kv, D), generator=g))
    q = torch.randn((T, Hq, D), generator=g).to(BF16)
    gt = torch.randn((T, Hq, 2 * D), generator=g).to(BF16) if gate else None
    cu = offsets(lens)
    tab = table.tolist()
    if edit is not None:
        edit(pool, q, tab)
    out = torch.full((T, Hq, D), 9.0, dtype=BF16, device=dev)
    gd = gt.to(dev) if gate else None
    pages = gpu_pool(pool, dev)
    paged.attention(pages, q.to(dev), i32(tab, dev), i32(pos, dev), max_keys, i32(cu, dev), max_rows,
                    gd[..., D:] if gate else None, scale, out, keys_per_split=kps)
    want, tol = ref.attention(pool, q, tab, pos, cu, gt[..., D:] if gate else None, scale, fill=9.0,
                              terms=2 if min(max_rows or T, T) <= 8 else 1)
    got = out.cpu().double()
    assert torch.equal(got.isfinite(), want.isfinite())
    fin = want.isfinite()
    far = (got - want).abs()[fin]
    assert bool((far <= tol[fin]).all()), f"{float((far - tol[fin]).max())} over at {float(far.max())}"
    return got, want


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv,page,lens,pos", [
    (256, 16, 4, 64, [1], [0]), (256, 16, 4, 64, [1], [700]), (256, 16, 4, 16, [4], [333]), (256, 8, 2, 32, [8], [127]),
    (128, 4, 2, 16, [1, 3, 0, 20], [0, 130, 50, 14]), (128, 8, 8, 64, [2, 1], [95, 31]), (128, 6, 2, 128, [5], [250]),
    (128, 24, 1, 16, [3], [40]), (256, 16, 1, 256, [40], [300]), (128, 4, 2, 32, [130, 1, 65], [0, 200, 63]),
    (256, 4, 4, 64, [70], [0]),
])
def test_attention(dev, fmt, D, Hq, n_kv, page, lens, pos):
    check_attention(dev, fmt, D, Hq, n_kv, page, lens, pos)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kps", [0, 1 << 20, 256])
@pytest.mark.parametrize("D,Hq,n_kv,page,lens,pos", [
    (256, 16, 4, 64, [20], [0]), (256, 8, 4, 16, [33], [190]), (256, 16, 1, 256, [40], [300]), (128, 4, 2, 32, [130, 1, 65], [0, 200, 63]),
    (128, 4, 4, 16, [70, 0, 9], [5, 40, 127]), (256, 4, 4, 64, [129], [64]), (128, 6, 2, 1024, [50], [1000]),
])
def test_attention_of_prompt_chunks(dev, fmt, kps, D, Hq, n_kv, page, lens, pos):
    """One split (a split length past every key) and many."""
    check_attention(dev, fmt, D, Hq, n_kv, page, lens, pos, kps=kps, gate=kps == 0, wide=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv,page,lens,wide", [
    (128, 4, 1, 16, [500] + [1, 0, 2] * 40, False),     # more tiles than the longest sequence gets blocks
    (128, 4, 2, 32, [70] + [1] * 63, False), (256, 4, 1, 16, [1] * 33 + [40] + [2] * 30, False),
    (128, 4, 1, 16, [600] + [3, 0, 9] * 13, True), (256, 8, 2, 64, [5, 0, 130, 1], True),
])
@pytest.mark.parametrize("bound", [False, True])
def test_attention_of_unequal_sequences(dev, fmt, D, Hq, n_kv, page, lens, wide, bound):
    pos = [(37 * b) % 90 for b in range(len(lens))]
    check_attention(dev, fmt, D, Hq, n_kv, page, lens, pos, wide=wide, max_rows=max(lens) if bound else None)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv,page,lens,pos,max_rows", [
    (256, 8, 4, 16, [1] * 24, [0, 700, 5, 127, 128, 300] * 4, 1),
    (128, 4, 2, 32, [1, 2, 0, 4] * 12, [0, 130, 50, 14, -1, -3, 400, 255] * 6, 4),
    (128, 8, 8, 64, [1] * 100, list(range(0, 300, 3)), 1),          # two rounds of the search
    (256, 16, 4, 64, [4] + [1] * 23, [900] + [0] * 23, 4),          # one sequence has nearly every step
    (128, 4, 2, 16, [1] * 20 + [23] + [1] * 30 + [9], [40] * 20 + [-6] + [60] * 30 + [200], 1),   # more rows than max_rows
    (128, 24, 8, 1024, [2] * 13, [0, -2, 1] * 4 + [1500], 2),
])
def test_attention_of_many_long_contexts(dev, fmt, D, Hq, n_kv, page, lens, pos, max_rows):
    """A bound on the keys far above them: the steps of all sequences in equal runs."""
    check_attention(dev, fmt, D, Hq, n_kv, page, lens, pos, gate=True, wide=True, max_rows=max_rows)


@pytest.mark.parametrize("fmt", FORMATS)
def test_graph_of_many_long_contexts(dev, fmt):
    """Replays at new positions, beside eager calls, and the same bits whenever it is called."""
    D, Hq, n_kv, page, B, W = 256, 8, 4, 64, 30, 64
    pages = paged.KVPages.alloc(B * W, n_kv, D, fmt, page, dev)
    for x in pages.tensors():
        if x.dtype == torch.float32:
            x.copy_(0.01 + torch.rand(x.shape, generator=gen(41)))
        elif fmt == "bf16":
            x.copy_(torch.randn(x.shape, generator=gen(42)))
        else:
            x.view(torch.uint8).copy_(torch.randint(0, 100, x.shape, generator=gen(43), dtype=torch.uint8))
    table = torch.randperm(B * W, generator=gen(44)).to(torch.int32).view(B, W).to(dev)
    q = torch.randn((B, Hq, D), generator=gen(45)).to(BF16).to(dev)
    pos = torch.randint(0, W * page, (B,), generator=gen(46)).to(torch.int32).to(dev)
    want = paged.attention(pages, q, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = paged.attention(pages, q, table, pos)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(paged.attention(pages, q, table, pos), want)
        pos.copy_(torch.randint(-1, W * page, (B,), generator=gen(50 + i)))
        one = paged.attention(pages, q[7:8], table[7:8], pos[7:8])
        want = paged.attention(pages, q, table, pos)
        assert torch.allclose(one[0].float(), want[7].float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(one.abs().max()))


def test_append_read_and_input_stage_of_unequal_sequences(dev):
    """Every row of a batch of one long and many short sequences, as in a call of its own."""
    D, Hq, n_kv, page, lens = 128, 4, 2, 16, [300] + [1, 0, 3] * 30 + [64]
    pos = [(5 * b) % 50 for b in range(len(lens))]
    T, cu = sum(lens), i32(offsets(lens), dev)
    table, n_pages = layout(lens, pos, page, 31)
    table, posd = i32(table.tolist(), dev), i32(pos, dev)
    proj = torch.randn((T, Hq * 2 * D + 2 * n_kv * D), generator=gen(32)).to(BF16).to(dev)
    w, freqs = torch.ones(D, dtype=BF16, device=dev), paged.rope_freqs(64, 1e6, dev)
    a, b, c = (paged.KVPages.alloc(n_pages, n_kv, D, "int8", page, dev) for _ in range(3))
    q = paged.attn_qk_rope(a, proj, w, w, table, posd, freqs, 1e-6, cu)
    kv = torch.randn((T, n_kv, D), generator=gen(33)).to(BF16).to(dev)
    paged.kv_append(c, kv, kv, table, posd, cu)
    k, _ = paged.kv_read(c, table, posd, T, cu)
    for s, n in enumerate(lens):
        if n:
            at = slice(sum(lens[:s]), sum(lens[:s + 1]))
            one = (table[s:s + 1].contiguous(), posd[s:s + 1])
            assert torch.equal(q[at], paged.attn_qk_rope(b, proj[at], w, w, *one, freqs, 1e-6))
            assert torch.equal(k[at], paged.kv_read(c, *one, n)[0])
    for x, y in zip(a.tensors(), b.tensors()):
        assert torch.equal(x, y)
    assert float((k.float() - kv.float()).abs().max()) <= float(kv.float().abs().max()) * (0.5 / 127 + 2.0 ** -8)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kps,max_keys", [(128, None), (256, 1200), (0, 1), (128, 130), (1152, None)])
def test_attention_splits(dev, fmt, kps, max_keys):
    """Any split, and a bound on the keys that is too small."""
    check_attention(dev, fmt, 128, 4, 2, 64, [2, 1, 9], [1100, 511, 256], kps=kps, max_keys=max_keys, gate=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_gate_scale_padding(dev, fmt):
    check_attention(dev, fmt, 256, 8, 4, 32, [3, 12], [77, 0], gate=True, scale=0.02, pad=4)
    check_attention(dev, fmt, 128, 4, 2, 16, [3, 40], [77, 0], max_rows=1, fill_gain=30.0)
    check_attention(dev, fmt, 256, 8, 4, 32, [3, 50], [77, 0], gate=True, scale=0.02, pad=4, wide=True)
    check_attention(dev, fmt, 128, 4, 2, 16, [3, 140], [77, 0], max_rows=33, fill_gain=30.0, wide=True)
    check_attention(dev, fmt, 128, 4, 2, 16, [3, 40], [77, 9], scale=0.0, wide=True)
    check_attention(dev, fmt, 128, 4, 2, 16, [3], [77], scale=0.0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("long", [False, True])
def test_attention_rows_that_see_nothing(dev, fmt, long):
    """Negative positions and pages that are not there; a row without any key gets zeros."""
    n = 70 if long else 6

    def edit(pool, q, tab):
        tab[0][0] = -1                          # the first page of sequence 0
        tab[2] = [99] * len(tab[2])

    if long:
        check_attention(dev, fmt, 128, 4, 2, 16, [n, n, n], [5, -4, 20], edit=edit, wide=True, kps=1 << 20)
        check_attention(dev, fmt, 128, 4, 2, 16, [n, n, n], [-100, -4, -69], edit=edit, wide=True, kps=1 << 20)
    got, _ = check_attention(dev, fmt, 128, 4, 2, 16, [n, n, n], [5, -4, 20], edit=edit, wide=long)
    assert bool((got[n:n + 4] == 0).all()) and bool((got[2 * n:3 * n] == 0).all()) and bool((got[:min(n, 11)] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv,n", [(256, 16, 4, 4), (128, 4, 2, 40), (256, 4, 2, 90), (128, 16, 1, 3), (128, 2, 2, 200),
                                         (256, 16, 4, 30)])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_nan_and_inf_stay_with_the_rows_that_see_them(dev, fmt, D, Hq, n_kv, n, wide):
    """A key or value that is not a number, seen by later rows only; a query that is not one."""
    pos = 61

    def edit(pool, q, tab):
        k, v = (torch.randn((n_kv, D), generator=gen(10 + i)) for i in range(2))
        k2, v2 = k.clone(), v.clone()
        v2[0, 3] = math.nan
        pool.put(pool.slot(tab[0], pos + n // 2), k, v2)
        v2 = v.clone()
        v2[-1, 7] = math.inf
        pool.put(pool.slot(tab[0], pos + n // 2 + 1), k2, v2)
        k2[0, 1] = math.nan
        pool.put(pool.slot(tab[0], pos + n - 1), k2, v)
        q[1, 0, 5] = math.nan

    _, want = check_attention(dev, fmt, D, Hq, n_kv, 16, [n], [pos], edit=edit, wide=wide)
    assert bool(want[0].isfinite().all()) and not bool(want[n - 1].isfinite().all())


def test_attention_strided_queries_and_workspace(dev):
    """q and gate as columns of projection rows (odd strides too), a caller's workspace, another stream."""
    D, Hq, n_kv, page, T, p = 128, 4, 2, 32, 5, 400
    pages = paged.KVPages(*(torch.randn((14, n_kv, page, D), device=dev).to(BF16) for _ in range(2)))
    table, pos = i32([list(range(13, -1, -1))], dev), i32([p], dev)
    proj = torch.randn((T, Hq * 2 * D + 3), device=dev).to(BF16)
    qg = proj[:, :Hq * 2 * D].unflatten(1, (Hq, 2 * D))
    q, gate = qg[..., :D], qg[..., D:]
    want = paged.attention(pages, q.contiguous(), table, pos, gate=gate.contiguous())
    need = paged.workspace_bytes(pages, 1, T, Hq, 14 * page)
    ws = torch.full(((need + 3) // 4,), math.nan, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged.attention(pages, q, table, pos, gate=gate, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_keep_their_bits_in_calls_of_up_to_8(dev, fmt):
    """At one keys_per_split a row's result does not depend on the rows it comes with."""
    D, Hq, n_kv, page, p = 256, 16, 4, 64, 900
    pages = paged.KVPages.alloc(16, n_kv, D, fmt, page, dev)
    table = i32([list(range(16))], dev)
    kv = torch.randn((p + 8, n_kv, D), generator=gen(12)).to(BF16).to(dev)
    paged.kv_append(pages, kv, kv.flip(0), table, i32([0], dev))
    q = torch.randn((8, Hq, D), generator=gen(13)).to(BF16).to(dev)
    whole = paged.attention(pages, q, table, i32([p], dev), keys_per_split=128)
    for i in range(8):
        one = paged.attention(pages, q[i:i + 1], table, i32([p + i], dev), keys_per_split=128)
        assert torch.equal(one[0], whole[i])
    two = paged.attention(pages, torch.cat([q[:3], q[4:5]]), i32([list(range(16))] * 2, dev), i32([p, p + 4], dev),
                          cu=i32([0, 3, 4], dev), keys_per_split=128)
    assert torch.equal(two[:3], whole[:3]) and torch.equal(two[3], whole[4])


@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_pool_past_32_bits(dev, fmt):
    """Pages whose bytes lie past 2^31 (and, in bf16, 2^32) of the pool."""
    D, n_kv, page, n = 256, 4, 64, 33000
    pages = paged.KVPages.alloc(n, n_kv, D, fmt, page, dev)
    T = 100
    kv = torch.randn((T, n_kv, D), generator=gen(14)).to(BF16).to(dev)
    q = torch.randn((T, 16, D), generator=gen(15)).to(BF16).to(dev)
    small = paged.KVPages.alloc(2, n_kv, D, fmt, page, dev)
    got = []
    for pg, tab in ((pages, [[n - 1, n - 3]]), (small, [[0, 1]])):
        t, p0 = i32(tab, dev), i32([0], dev)
        paged.kv_append(pg, kv, kv.flip(0), t, p0)
        got.append([*paged.kv_read(pg, t, p0, T), paged.attention(pg, q, t, p0),
                    paged.attention(pg, q, torch.cat([t, torch.full((1, 100), -1, dtype=torch.int32, device=dev)], 1), p0),
                    paged.attention(pg, q[-1:], t, i32([T - 1], dev))])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
def test_graph_of_the_decode_step(dev, fmt):
    """Append, attention and read-back captured once and replayed at other positions, tables and
    values, with eager work between the replays; two graphs on the same pages."""
    D, Hq, n_kv, page, B, W = 256, 8, 4, 32, 3, 20
    pages = paged.KVPages.alloc(B * W, n_kv, D, fmt, page, dev)
    table = torch.randperm(B * W, generator=gen(16)).to(torch.int32).view(B, W).to(dev)
    pos = i32([0, 0, 0], dev)
    kv = torch.randn((B, 600, n_kv, D), generator=gen(17)).to(BF16).to(dev)
    held = [300, 17, 500]
    cu = i32(offsets(held), dev)
    rows = torch.cat([kv[b, :n] for b, n in enumerate(held)])
    paged.kv_append(pages, rows, rows.flip(0), table, pos, cu)
    pos.copy_(i32(held, dev))
    k, q = torch.empty((B, n_kv, D), dtype=BF16, device=dev), torch.empty((B, Hq, D), dtype=BF16, device=dev)

    def step():
        paged.kv_append(pages, k, k, table, pos)
        return paged.attention(pages, q, table, pos), *paged.kv_read(pages, table, pos, B)

    k.zero_()
    q.zero_()
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for i in range(6):
        k.copy_(kv[:, 500 + i])
        q.copy_(torch.randn((B, Hq, D), generator=gen(20 + i)).to(BF16))
        g, outs = graphs[i % 2]
        for o in outs:
            o.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        pos += 1
        if i == 2:
            table.copy_(table.flip(1))
            table[:, :W] = table.flip(1)


def test_empty_calls(dev):
    pages = paged.KVPages.alloc(2, 2, 128, "int8", 16, dev)
    e = torch.empty((0, 2, 128), dtype=BF16, device=dev)
    table, pos = i32([[0, 1]], dev), i32([0], dev)
    paged.kv_append(pages, e, e, table, pos)
    assert paged.attention(pages, e, table, pos).shape == (0, 2, 128)
    assert paged.kv_read(pages, table, pos, 0)[0].shape == (0, 2, 128)
    cu = i32([0, 0], dev)
    out = torch.full((3, 2, 128), 4.0, dtype=BF16, device=dev)
    q = torch.randn((3, 2, 128), device=dev).to(BF16)
    paged.attention(pages, q, table, pos, cu=cu, out=out)
    assert bool((out == 4.0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv", [(256, 16, 4), (128, 4, 2)])
def test_a_prompt_and_its_decode_steps(dev, fmt, D, Hq, n_kv):
    """The operators as they are used: a prompt in chunks and single tokens after it through the input stage
    and attention, against the same on rows kept dense."""
    page, n = 32, 150
    T = n + 4
    width = Hq * 2 * D + 2 * n_kv * D
    proj = torch.randn((T, width), generator=gen(30)).to(BF16)
    w = (1.0 + 0.1 * torch.randn(D, generator=gen(31))).to(BF16)
    pages = paged.KVPages.alloc(8, n_kv, D, fmt, page, dev)
    table = [[5, 2, 7, 0, 3, -1]]
    freqs = paged.rope_freqs(32, 1e6, dev)
    pd, wd, td = proj.to(dev), w.to(dev), i32(table, dev)
    outs, qs = [], []
    for lo, hi in ((0, 64), (64, 127), (127, n), *((i, i + 1) for i in range(n, T))):
        pos = i32([lo], dev)
        q = paged.attn_qk_rope(pages, pd[lo:hi], wd, wd, td, pos, freqs, 1e-6)
        gate = pd[lo:hi, :Hq * 2 * D].unflatten(1, (Hq, 2 * D))[..., D:]
        outs.append(paged.attention(pages, q, td, pos, hi, gate=gate))
        qs.append(q)
    pool = ref.Pool(8, n_kv, page, D, fmt)
    pool.k, pool.v = pages.k.cpu(), pages.v.cpu()
    if fmt != "bf16":
        pool.ks, pool.vs = pages.k_scale.cpu(), pages.v_scale.cpu()
    q, gate = torch.cat(qs).cpu(), proj[:, :Hq * 2 * D].unflatten(1, (Hq, 2 * D))[..., D:]
    want, tol = ref.attention(pool, q, table, [0], None, gate, terms=1)
    assert bool(((torch.cat(outs).cpu().double() - want).abs() <= tol).all())
    wq, wk, wv = ref.qk_rope(proj, w, w, Hq, n_kv, D, freqs.cpu(), 1e-6, torch.arange(T))
    assert bool(((q.double() - wq).abs() <= 2.0 ** -8 * wq.abs() + 2.0 ** -19 * wq.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("T,kps", [(1, 0), (4, 0), (4, 256), (40, 0)])
def test_one_workspace_for_a_growing_context(dev, T, kps):
    """A buffer made once for the longest context serves every shorter bound, with the bits of a buffer of the call's own."""
    D, Hq, n_kv, page = 256, 16, 4, 64
    pages = paged.KVPages.alloc(320, n_kv, D, "int8", page, dev)
    table, pos = i32([list(range(320))], dev), i32([0], dev)
    kv = torch.randn((20480, n_kv, D), generator=gen(60)).to(BF16).to(dev)
    paged.kv_append(pages, kv, kv.flip(0), table, pos)
    q = torch.randn((T, Hq, D), generator=gen(61)).to(BF16).to(dev)
    ws = torch.empty(paged.workspace_bytes(pages, 1, T, Hq, 20000, keys_per_split=kps), dtype=torch.uint8, device=dev)
    for keys in (20000, 16384, 9000, 8192, 3000, 300, T):
        pos.fill_(keys - T)
        a = paged.attention(pages, q, table, pos, keys, keys_per_split=kps, workspace=ws)
        assert torch.equal(a, paged.attention(pages, q, table, pos, keys, keys_per_split=kps))


@pytest.fixture()
def two_terms(monkeypatch):
    """The reference's tolerance for weights of two bf16 terms, whatever the number of rows."""
    plain = ref.attention
    monkeypatch.setattr(ref, "attention", lambda *a, **kw: plain(*a, **{**kw, "terms": 2}))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,Hq,n_kv,page,lens,pos,kps", [
    (256, 16, 1, 256, [40], [300], 0), (128, 4, 2, 32, [130, 1, 65], [0, 200, 63], 0), (256, 4, 4, 64, [70], [0], 1 << 20),
    (128, 4, 4, 16, [70, 0, 9], [5, 40, 127], 256), (256, 8, 4, 16, [33], [190], 1 << 20), (256, 16, 4, 64, [20], [0], 0),
])
def test_weights_keep_two_terms_in_calls_of_many_rows(dev, two_terms, fmt, wide, D, Hq, n_kv, page, lens, pos, kps):
    """Both forms that serve more than 8 rows, of few rows and of prompt chunks (wide), hold a weight in 16 bits."""
    check_attention(dev, fmt, D, Hq, n_kv, page, lens, pos, kps=kps, gate=kps == 0, wide=wide)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,n_kv", [(256, 8, 4), (128, 8, 2)])
def test_prompt_chunk_whose_scores_rise(dev, two_terms, fmt, D, Hq, n_kv):
    """Scores that grow along the keys move the reference in every step, between a tile's weights and their terms too."""
    def edit(pool, q, tab):
        q.fill_(0.0)
        q[:, :, 0] = 1.0
        for x in range(300):
            j, s = pool.slot(tab[0], x)
            k = pool.k[j, :, s].float() * 0.125
            k[:, 0] = float(x if x % 7 else x - 40) * 4.0
            v = pool.get((j, s))[1]
            pool.put((j, s), k if fmt == "bf16" else k.clamp(-2000, 2000), v)

    check_attention(dev, fmt, D, Hq, n_kv, 16, [100], [200], edit=edit, wide=True, scale=0.5)
    check_attention(dev, fmt, D, Hq, n_kv, 16, [100], [200], edit=edit, wide=True, scale=0.5, kps=1 << 20, gate=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,B,width,kps", [
    (1, 3, 4, 0), (6, 3, 4, 1 << 20), (6, 6, 20, 128), (80, 3, 3000, 1 << 20), (80, 3, 3000, 0), (1, 48, 300, 0), (3, 48, 300, 0),
])
def test_rows_that_see_nothing_are_zero_whatever_their_gate(dev, fmt, n, B, width, kps):
    """Rows before position 0 and of sequences without pages: a gate that is NaN there changes no bit of any row, in
    every form (one split, merged splits, chunks, runs of steps)."""
    D, Hq, n_kv, page = 128, 4, 2, 16
    held = [(-4, 9, 5)[b % 3] for b in range(B)]
    need = [0 if b % 3 == 2 else -(-(p + n) // page) if p + n > 0 else 0 for b, p in enumerate(held)]
    pages = paged.KVPages.alloc(max(1, sum(need)), n_kv, D, fmt, page, dev)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = torch.arange(at, at + m)
        at += m
    table = table.to(dev)
    kv = torch.randn((B * page * 6, n_kv, D), generator=gen(70)).to(BF16).to(dev)
    paged.kv_append(pages, kv, kv.flip(0), table, i32([0] * B, dev))
    q = torch.randn((B * n, Hq, D), generator=gen(71)).to(BF16).to(dev)
    gate = torch.randn((B * n, Hq, D), generator=gen(72)).to(BF16).to(dev)
    blind = torch.tensor([b % 3 == 2 or p + i < 0 for b, p in enumerate(held) for i in range(n)], device=dev)
    bad = gate.clone()
    bad[blind] = math.nan
    cu = i32([n * b for b in range(B + 1)], dev)
    for rows in (None, cu):
        kw = {"cu": rows, "max_rows": n} if rows is not None else {}
        a = paged.attention(pages, q, table, i32(held, dev), gate=gate, keys_per_split=kps, **kw)
        for _ in range(3):
            got = paged.attention(pages, q, table, i32(held, dev), gate=bad, keys_per_split=kps, **kw)
            assert torch.equal(a, got) and bool((got[blind] == 0).all()) and bool((got[~blind] != 0).any())


@pytest.mark.parametrize("fmt", FORMATS)
def test_graph_after_its_table_was_rewritten(dev, fmt):
    """A captured step replayed after every sequence has moved to other pages, twice, beside the eager step."""
    D, Hq, n_kv, page, B, W = 128, 4, 2, 16, 3, 12
    pages = paged.KVPages.alloc(2 * B * W, n_kv, D, fmt, page, dev)
    perm = torch.randperm(2 * B * W, generator=gen(80)).to(torch.int32)
    table = perm[:B * W].view(B, W).to(dev)
    pos = i32([0] * B, dev)
    held = [100, 17, 150]
    kv = torch.randn((B, 200, n_kv, D), generator=gen(81)).to(BF16).to(dev)
    rows, cu = torch.cat([kv[b, :n] for b, n in enumerate(held)]), i32(offsets(held), dev)
    k, q = torch.empty((B, n_kv, D), dtype=BF16, device=dev), torch.empty((B, Hq, D), dtype=BF16, device=dev)

    def step():
        paged.kv_append(pages, k, k, table, pos)
        return paged.attention(pages, q, table, pos), *paged.kv_read(pages, table, pos, B)

    def fill():
        pos.zero_()
        paged.kv_append(pages, rows, rows.flip(0), table, pos, cu)
        pos.copy_(i32(held, dev))

    k.zero_()
    q.zero_()
    fill()
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for i in range(4):
        old = table.clone()
        at = torch.arange(B * W) + (0, B * W, 5, 31)[i]
        table.copy_(perm[at % (2 * B * W)].view(B, W).roll(i, 0))
        assert i == 0 or not bool((table == old).any())
        for x in pages.tensors():
            x.view(torch.uint8).zero_()
        fill()
        for j in range(2):
            k.copy_(kv[:, 180 + i + j])
            q.copy_(torch.randn((B, Hq, D), generator=gen(82 + 2 * i + j)).to(BF16))
            for o in outs:
                o.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            want = step()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            assert bool((outs[0] != 0).all()) and bool((outs[1] != 0).any())
            pos += 1


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_keep_their_bits_in_large_ragged_calls_of_up_to_8(dev, fmt):
    """With max_rows given, sequences of up to 8 rows in a call large enough for the chunk form, against calls of their own."""
    D, Hq, n_kv, page, B, n = 128, 8, 2, 16, 20, 700
    pages = paged.KVPages.alloc(B * 50, n_kv, D, fmt, page, dev)
    table = torch.randperm(B * 50, generator=gen(90)).to(torch.int32).view(B, 50).to(dev)
    kv = torch.randn((B * 750, n_kv, D), generator=gen(91)).to(BF16).to(dev)
    paged.kv_append(pages, kv, kv.flip(0), table, i32([0] * B, dev))
    lens = [8 if b % 4 else 1 + b % 7 for b in range(B)]
    pos = i32([n - 13 * b for b in range(B)], dev)
    cu, T = offsets(lens), sum(lens)
    q = torch.randn((T, Hq, D), generator=gen(92)).to(BF16).to(dev)
    wide = torch.cat([table, torch.full((B, 1000), -1, dtype=torch.int32, device=dev)], 1)
    assert T * Hq * 1050 * page * D > 1.28e9
    whole = paged.attention(pages, q, wide, pos, cu=i32(cu, dev), max_rows=8, keys_per_split=256)
    for b in range(B):
        for i in (0, lens[b] - 1):
            one = paged.attention(pages, q[cu[b] + i:cu[b] + i + 1], table[b:b + 1], pos[b:b + 1] + i, keys_per_split=256)
            assert torch.equal(one[0], whole[cu[b] + i])
