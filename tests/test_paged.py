"""Paged KV cache on the CPU: what the entry points and their front end refuse, before any GPU work."""

import ctypes
import gc

import pytest
import torch

from qvex import _C, paged

BF16 = torch.bfloat16


@pytest.fixture()
def buf():
    b = ctypes.create_string_buffer(1 << 12)
    yield (ctypes.addressof(b) + 15) // 16 * 16
    del b


def pages_of(p, **kw):
    f = {"k": p, "v": p, "k_scales": p, "v_scales": p, "n_pages": 4, "page": 64, "Hkv": 2, "D": 128, "format": 1, **kw}
    return _C.KvPages(*f.values())


def rows_of(p, **kw):
    f = {"table": p, "pos": p, "cu": p, "table_stride": 4, "table_width": 4, "B": 2, "L": 3, "T": 5, **kw}
    return _C.KvRows(*f.values())


def calls(p, pages, rows):
    """Every entry point on these structs."""
    a, b = ctypes.byref(pages), ctypes.byref(rows)
    return {"qvex_paged_append": (a, b, p, 256, 128, p, 256, 128, None),
            "qvex_paged_qk_rope": (a, b, p, 4 * 2 * 128 + 4 * 128, p, p, 4, 32, p, 1e-6, p, None),
            "qvex_paged_read": (a, b, p, p, 0, None),
            "qvex_paged_attention": (a, b, p, 512, 128, 4, 100, 0, None, 0, 0, 0.1, p, p, 1 << 30, None)}


@pytest.mark.parametrize("kw,match", [
    ({"format": 3}, "format"), ({"format": -1}, "format"), ({"D": 64}, "D=64"), ({"page": 48}, "page=48"),
    ({"page": 8}, "page=8"), ({"page": 2048}, "page=2048"), ({"n_pages": 0}, "n_pages"), ({"Hkv": 0}, "Hkv=0"),
    ({"k": None}, "16-byte"), ({"v_scales": None}, "scales"),
])
def test_every_entry_point_refuses_bad_pages(buf, kw, match):
    for name, args in calls(buf, pages_of(buf, **kw), rows_of(buf)).items():
        with pytest.raises(_C.QvexError, match=f"{name}.*{match}"):
            _C.call(name, *args)


def test_every_entry_point_refuses_misaligned_pages(buf):
    for name, args in calls(buf, pages_of(buf, k=buf + 8), rows_of(buf)).items():
        with pytest.raises(_C.QvexError, match="16-byte"):
            _C.call(name, *args)


@pytest.mark.parametrize("kw,match", [
    ({"B": 0}, "B=0"), ({"B": 70000}, "B=70000"), ({"L": 0}, "L=0"), ({"T": -1}, "T=-1"), ({"T": 1 << 30}, "T="),
    ({"cu": None}, "T=5"), ({"table": None}, "table"), ({"pos": None}, "positions"), ({"table_width": 0}, "table_width"),
    ({"table_stride": 3}, "table_stride"), ({"table_width": 1 << 25, "table_stride": 1 << 25}, "table_width"),
])
def test_every_entry_point_refuses_bad_rows(buf, kw, match):
    for name, args in calls(buf, pages_of(buf), rows_of(buf, **kw)).items():
        with pytest.raises(_C.QvexError, match=f"{name}.*{match}"):
            _C.call(name, *args)


def test_null_structs_are_refused(buf):
    for name, args in calls(buf, pages_of(buf), rows_of(buf)).items():
        with pytest.raises(_C.QvexError, match="null"):
            _C.call(name, None, *args[1:])
        with pytest.raises(_C.QvexError, match="null"):
            _C.call(name, args[0], None, *args[2:])


def edited(args, **at):
    out = list(args)
    for i, v in at.items():
        out[int(i[1:])] = v
    return out


@pytest.mark.parametrize("name,at,match", [
    ("qvex_paged_append", {"_2": None}, "null"), ("qvex_paged_append", {"_5": None}, "null"),
    ("qvex_paged_qk_rope", {"_2": None}, "null"), ("qvex_paged_qk_rope", {"_3": 100}, "p_stride"),
    ("qvex_paged_qk_rope", {"_6": 3}, "Hq=3"), ("qvex_paged_qk_rope", {"_7": 33}, "rot_dim"),
    ("qvex_paged_qk_rope", {"_7": 130}, "rot_dim"), ("qvex_paged_qk_rope", {"_8": None}, "null"),
    ("qvex_paged_read", {"_2": None}, "aligned"), ("qvex_paged_attention", {"_2": None}, "null"),
    ("qvex_paged_attention", {"_5": 5}, "Hq=5"), ("qvex_paged_attention", {"_6": 0}, "max_keys"),
    ("qvex_paged_attention", {"_7": 100}, "keys_per_split"), ("qvex_paged_attention", {"_7": -128}, "keys_per_split"),
    ("qvex_paged_attention", {"_6": 5000, "_7": 128, "_14": 1000}, "workspace"),
    ("qvex_paged_attention", {"_6": 5000, "_7": 128, "_13": None}, "workspace"), ("qvex_paged_attention", {"_12": None}, "null"),
])
def test_bad_arguments_are_refused(buf, name, at, match):
    args = edited(calls(buf, pages_of(buf), rows_of(buf))[name], **at)
    with pytest.raises(_C.QvexError, match=match):
        _C.call(name, *args)


def test_workspace_bytes():
    f = _C.lib().qvex_paged_attention_workspace_bytes
    assert f(2, 3, 5, 4, 2, 128, 100, 0) == 0                       # one split
    assert f(1, 1, 1, 16, 4, 256, 4096, 128) == 16 * 32 * 258 * 4
    assert f(1, 1, 1, 16, 3, 256, 4096, 128) == 0 and f(1, 1, 1, 16, 4, 64, 4096, 128) == 0     # refused shapes
    # a workspace of a call serves calls of fewer keys
    for kps in (0, 128, 512):
        sizes = [f(3, 4, 9, 8, 2, 128, mk, kps) for mk in range(1, 5000, 77)]
        assert kps == 0 or sizes == sorted(sizes)


def test_front_end_refuses_bad_pools_and_host_memory():
    k, s = torch.zeros((2, 2, 16, 128), dtype=torch.int8), torch.zeros((2, 2, 16))
    for args, match in (((k.float(), k.float()), "bf16, int8"), ((k, k), "need k_scale"), ((k, k[:1], s, s), "differ"),
                        ((k, k.to(BF16), s, s), "v pages"), ((k, k, s, s.double()), "v_scale"),
                        ((k, k, s, s[:1]), "v_scale"), ((k.to(BF16), k.to(BF16), s), "no scales"),
                        ((k[..., :64].contiguous(), k[..., :64].contiguous(), s, s), "heads of 128 or 256"),
                        ((k[:, :, :8].contiguous(), k[:, :, :8].contiguous(), s[..., :8].contiguous(),
                          s[..., :8].contiguous()), "power of two")):
        with pytest.raises(_C.QvexError, match=match):
            paged.KVPages(*args)
    with pytest.raises(_C.QvexError, match="unknown KV format"):
        paged.KVPages.alloc(2, 2, 128, "int4")
    x, t, p = torch.zeros((1, 2, 128), dtype=BF16), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(_C.QvexError, match="must be on a GPU"):
        paged.kv_append(paged.KVPages(k, k, s, s), x, x, t, p)


class _FakePages(paged.KVPages):
    """A handle over host memory, for the checks that run before a launch."""

    def __init__(self):
        self.fmt, self.n_pages, self.n_kv, self.page, self.head_dim = "int8", 4, 2, 16, 128
        self.device = torch.device("cpu")
        self._c = None

    def _stream(self):
        raise AssertionError("a refused call reached the launch")


def good():
    z = torch.zeros
    return {"x": z((6, 2, 128), dtype=BF16), "table": z((2, 4), dtype=torch.int32), "pos": z(2, dtype=torch.int32),
            "cu": torch.tensor([0, 2, 6], dtype=torch.int32), "proj": z((6, 4 * 2 * 128 + 4 * 128), dtype=BF16),
            "w": z(128, dtype=BF16), "freqs": z(16, dtype=torch.float64)}


@pytest.mark.parametrize("key,value,match", [
    ("x", torch.zeros((6, 2, 128)), "bf16"), ("x", torch.zeros((6, 3, 128), dtype=BF16), "kv heads|must be bf16"),
    ("x", torch.zeros((6, 2, 64), dtype=BF16), "128"), ("x", torch.zeros((6, 2, 256), dtype=BF16)[..., ::2], "consecutive"),
    ("table", torch.zeros((2, 4)), "table"), ("table", torch.zeros((3, 4), dtype=torch.int32), "table"),
    ("table", torch.zeros((2, 8), dtype=torch.int32)[:, ::2], "table"), ("pos", torch.zeros(2), "pos"),
    ("pos", torch.zeros((2, 1), dtype=torch.int32), "pos"), ("cu", torch.zeros(2, dtype=torch.int32), "cu"),
    ("cu", torch.zeros(3, dtype=torch.int64), "cu"),
])
def test_front_end_refuses_bad_tensors(key, value, match):
    a = {**good(), key: value}
    pages = _FakePages()
    with pytest.raises(_C.QvexError, match=match):
        paged.kv_append(pages, a["x"], a["x"], a["table"], a["pos"], a["cu"])
    with pytest.raises(_C.QvexError, match=match):
        paged.attention(pages, a["x"], a["table"], a["pos"], cu=a["cu"])
    if key != "x":
        with pytest.raises(_C.QvexError, match=match):
            paged.kv_read(pages, a["table"], a["pos"], 6, a["cu"])
        with pytest.raises(_C.QvexError, match=match):
            paged.attn_qk_rope(pages, a["proj"], a["w"], a["w"], a["table"], a["pos"], a["freqs"], 1e-6, a["cu"])


@pytest.mark.parametrize("key,value,match", [
    ("proj", torch.zeros((6, 1000), dtype=BF16), "rows of 1000"), ("proj", torch.zeros((6, 1536)), "proj"),
    ("w", torch.zeros(64, dtype=BF16), "norm"), ("freqs", torch.zeros(16), "fp64"),
])
def test_front_end_refuses_bad_input_stage(key, value, match):
    a = {**good(), key: value}
    with pytest.raises(_C.QvexError, match=match):
        paged.attn_qk_rope(_FakePages(), a["proj"], a["w"], a["w"], a["table"], a["pos"], a["freqs"], 1e-6, a["cu"])


def test_front_end_refuses_rows_without_offsets():
    a = good()
    with pytest.raises(_C.QvexError, match="do not divide"):
        paged.kv_append(_FakePages(), a["x"][:5], a["x"][:5], a["table"], a["pos"])
    with pytest.raises(_C.QvexError, match="bf16 or fp32"):
        paged.kv_read(_FakePages(), a["table"], a["pos"], 6, dtype=torch.float16)
    with pytest.raises(_C.QvexError, match="out must"):
        paged.attention(_FakePages(), a["x"], a["table"], a["pos"], out=torch.zeros((6, 2, 128)))


# ---------------------------------------------------------------- pages handed to sequences

def fill(pool):
    """Every page's bytes name the page."""
    for j in range(pool.pages.n_pages):
        for x in pool.pages.tensors():
            x[j] = j % 100 + 1


def test_pool_takes_shares_and_gives():
    pool = paged.PagePool(4, 2, 128, "int8", 16, "cpu")
    a = pool.take(3)
    assert sorted(a) == [0, 1, 2] and pool.free == [3]
    pool.share(a[:1])
    pool.give(a)
    assert sorted(pool.free) == [1, 2, 3] and pool.holders == [1, 0, 0, 0]
    with pytest.raises(_C.QvexError, match="3 free pages of 4, 5"):
        pool.take(5)
    assert sorted(pool.free) == [1, 2, 3]
    pool.give(a[:1])
    assert len(pool.free) == 4


@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_pool_grows_and_keeps_its_pages(fmt):
    pool = paged.PagePool(2, 2, 128, fmt, 16, "cpu", growable=True)
    fill(pool)
    old = [x.clone() for x in pool.pages.tensors()]
    got = pool.take(5)
    assert len(set(got)) == 5 and pool.pages.n_pages >= 5
    for a, b in zip(pool.pages.tensors(), old):
        assert torch.equal(a[:2], b)


def test_workspace_of_many_long_contexts():
    """Runs of steps: a record of a tile for each of the runs and sequences of a kv head."""
    f = _C.lib().qvex_paged_attention_workspace_bytes
    assert f(64, 1, 64, 16, 4, 256, 8192, 0) == 4 * (64 + 64) * 16 * 258 * 4
    assert f(30, 2, 60, 32, 8, 128, 8192, 0) == 8 * (64 + 30) * 16 * 130 * 4
    assert f(64, 1, 64, 16, 4, 256, 8192, 8192 + 128) == 0          # a split length given: its splits
    assert f(64, 1, 64, 16, 4, 256, 128, 0) == 0


def test_workspace_of_a_call_with_and_without_row_offsets():
    """max_rows left out: enough for T / B rows each and for all of them in one sequence."""
    pages = paged.KVPages.alloc(64, 4, 256, "int8", 64, "cpu")
    f = _C.lib().qvex_paged_attention_workspace_bytes
    for B, T, mk in ((1, 1, 4000), (8, 64, 4000), (64, 64, 2000), (3, 100, 4000), (4, 512, 4096)):
        got = paged.workspace_bytes(pages, B, T, 16, mk)
        assert got == max(f(B, L, T, 16, 4, 256, mk, 0) for L in (max(T // B, 1), T))
    assert paged.workspace_bytes(pages, 4, 0, 16, 100) == 0


def test_cache_grows_without_moving_and_returns_its_pages():
    pool = paged.PagePool(40, 2, 128, "fp8", 16, "cpu")
    c = paged.PagedKVCache(pool, capacity=100)
    assert c.capacity == 256 and len(pool.free) == 24
    first = c.table[0, :16].clone()
    c.offset = 250
    assert not c.grow(256) and c.grow(257) and c.capacity == 512
    assert torch.equal(c.table[0, :16], first) and c.table[0].tolist() == c.ids
    with pytest.raises(_C.QvexError, match="free pages"):
        c.grow(1000)
    c.counters.graph_mode = True
    with pytest.raises(_C.QvexError, match="captured cycle"):
        c.grow(600)
    with pytest.raises(_C.QvexError, match="captured cycle"):
        c.rollback(1)
    c.counters.graph_mode = False
    del c
    assert len(pool.free) == 40 and not any(pool.holders)


def test_pool_does_not_move_under_a_captured_cycle():
    pool = paged.PagePool(16, 2, 128, "int8", 16, "cpu", growable=True)
    a = paged.PagedKVCache(pool, capacity=256)
    a.counters.graph_mode = True
    with pytest.raises(_C.QvexError, match="captured cycle drives a cache of this page pool"):
        paged.PagedKVCache(pool, capacity=256)
    a.counters.graph_mode = False
    paged.PagedKVCache(pool, capacity=256)


@pytest.mark.parametrize("at", [0, 1, 15, 16, 40, 255, 256, 300])
def test_clone_shares_the_prefix_and_an_append_never_writes_a_shared_page(at):
    pool = paged.PagePool(200, 2, 128, "int8", 16, "cpu")
    fill(pool)
    a = paged.PagedKVCache(pool, capacity=512)
    a.offset = at
    b = a.clone()
    n = at // 16
    assert b.offset == at and b.ids[:n] == a.ids[:n] and not set(b.ids[n:]) & set(a.ids)
    assert b.capacity > at and b.table[0].tolist() == b.ids
    if at % 16:      # the page that the next key goes to has the prefix's bytes
        for x in pool.pages.tensors():
            assert torch.equal(x[b.ids[n]], x[a.ids[n]])
    for c in (a, b):
        assert all(pool.holders[j] == 1 for j in c.ids[c.offset // 16:])
    # rolled back into the shared part, a cache takes pages of its own, with what they held
    if at > 20:
        held = list(a.ids)
        a.rollback(20)
        m = a.offset // 16
        assert a.ids[:m] == held[:m] and all(pool.holders[j] == 1 for j in a.ids[m:])
        assert b.ids[:n] == held[:n] and not set(a.ids[m:]) & set(b.ids)
        assert a.table[0, :len(a.ids)].tolist() == a.ids
        if a.offset % 16:
            for x in pool.pages.tensors():
                assert torch.equal(x[a.ids[m]], x[held[m]])
    c = b.clone()
    assert pool.holders == [sum(j in x.ids for x in (a, b, c)) for j in range(200)]
    del a, b, c
    assert len(pool.free) == 200 and not any(pool.holders)


def test_clone_of_layer_caches_shares_one_table_of_counters():
    from qvex.model import CacheCounters, LayerCaches
    pool = paged.PagePool(64, 2, 128, "int8", 64, "cpu")
    counters = CacheCounters(2, "cpu")
    caches = LayerCaches([paged.PagedKVCache(pool, counters, i, capacity=256) for i in range(2)], counters)
    for c in caches:
        c.offset = 130
    twin = caches.clone()
    assert twin[0].counters is twin[1].counters is twin.counters and twin.counters is not counters
    twin[0].offset = 131
    assert caches[0].offset == 130 and twin[1].offset == 130
    assert twin[0].pos.data_ptr() == twin.counters.ptr(0) and caches[1].pos.data_ptr() == counters.ptr(1)


@pytest.mark.parametrize("rotary_dim", [32, 0])
def test_attention_layer_has_its_frequencies_before_any_call(monkeypatch, rotary_dim):
    """A layer's first call may be inside a graph capture, where none can be made."""
    from qvex.model import Attention, Config, QLinear
    monkeypatch.setattr(QLinear, "fuse", staticmethod(lambda layers: None))
    cfg = Config.tiny()
    cfg.rotary_dim = rotary_dim
    w = torch.ones(cfg.head_dim, dtype=BF16)
    layer = Attention(cfg, {**dict.fromkeys(("q_proj", "k_proj", "v_proj", "o_proj")), "q_norm": w, "k_norm": w})
    if rotary_dim:
        assert torch.equal(layer._freqs, paged.rope_freqs(32, cfg.rope_theta, "cpu"))
    else:
        assert layer._freqs is None


def shared_pair(free, growable=False, n_pages=32):
    """A cache at 100 of pages of 16, its clone, and `free` pages left in their pool."""
    pool = paged.PagePool(n_pages, 2, 128, "int8", 16, "cpu", growable=growable)
    fill(pool)
    a = paged.PagedKVCache(pool, capacity=256)
    a.offset = 100
    b = a.clone()
    kept = pool.take(len(pool.free) - free)
    fill(pool)
    return pool, a, b, kept


def state_of(pool, *caches):
    return (list(pool.holders), sorted(pool.free), [t.clone() for t in pool.pages.tensors()],
            [(list(c.ids), c.offset, c.table.tolist()) for c in caches])


def assert_same(x, y):
    assert x[0] == y[0] and x[1] == y[1] and x[3] == y[3] and all(torch.equal(s, t) for s, t in zip(x[2], y[2]))


@pytest.mark.parametrize("to,free", [(30, 2), (30, 4), (0, 5), (80, 0), (7, 5)])
def test_a_rollback_without_pages_changes_nothing(to, free):
    """From 100 back to `to`: pages to // 16 .. 5 are shared, and more of them than are free (page 6 is
    the cache's own)."""
    pool, a, b, kept = shared_pair(free)
    need = 6 - to // 16
    before = state_of(pool, a, b)
    with pytest.raises(_C.QvexError, match=f"{free} free pages of 32, {need} are needed"):
        a.rollback(100 - to)
    assert_same(before, state_of(pool, a, b))
    pool.give(kept[:need - free])
    ids = list(a.ids)
    a.rollback(100 - to)                      # with enough of them
    first = to // 16
    assert a.offset == to and a.ids[:first] == ids[:first] and not set(a.ids[first:6]) & set(b.ids)
    assert a.table[0, :len(a.ids)].tolist() == a.ids and b.ids == before[3][1][0]
    if to % 16:
        for t in pool.pages.tensors():
            assert torch.equal(t[a.ids[first]], t[b.ids[first]])


def test_a_rollback_that_a_captured_cycle_forbids_to_grow_changes_nothing():
    pool, a, b, _ = shared_pair(1, growable=True)
    b.counters.graph_mode = True
    before = state_of(pool, a, b)
    with pytest.raises(_C.QvexError, match="captured cycle drives"):
        a.rollback(70)
    assert_same(before, state_of(pool, a, b))
    b.counters.graph_mode = False
    a.rollback(70)
    assert a.offset == 30 and pool.pages.n_pages > 32 and not set(a.ids[1:]) & set(b.ids)


def test_a_clone_that_fails_returns_its_pages(monkeypatch):
    pool, a, b, _ = shared_pair(14, n_pages=64)
    before = state_of(pool, a, b)

    def fails(*_):
        raise MemoryError

    monkeypatch.setattr(pool, "copy", fails)
    with pytest.raises(MemoryError):
        a.clone()
    gc.collect()
    assert before[0] == pool.holders and before[1] == sorted(pool.free)


@pytest.mark.parametrize("B,L,T,Hq,Hkv,D", [
    (1, 1, 1, 16, 4, 256), (1, 4, 4, 16, 4, 256), (3, 4, 9, 8, 2, 128), (24, 8, 192, 16, 4, 256), (64, 1, 64, 16, 4, 256),
    (30, 2, 60, 32, 8, 128), (40, 8, 320, 16, 4, 256), (1, 64, 64, 16, 4, 256), (1, 512, 512, 16, 4, 256),
    (12, 100, 1200, 4, 2, 128), (2, 9, 11, 24, 1, 128), (100, 30, 200, 4, 1, 128), (255, 2, 300, 16, 1, 256),
    (1, 40, 40, 32, 8, 128), (5, 17, 80, 6, 6, 256),
])
def test_a_workspace_serves_every_call_of_fewer_keys(B, L, T, Hq, Hkv, D):
    """The bytes of a call whose splits are chosen for it never fall as its keys grow, over every form it may take."""
    f = _C.lib().qvex_paged_attention_workspace_bytes
    keys = [*range(1, 6000, 37), *(128 * s + e for s in range(1, 400) for e in (0, 1)), *range(60000, 1 << 20, 40961)]
    sizes = [f(B, L, T, Hq, Hkv, D, mk, 0) for mk in sorted(keys)]
    assert sizes == sorted(sizes)


def test_workspace_bytes_with_max_rows_covers_calls_without_row_offsets():
    """max_rows bounds a ragged call's rows only; without offsets every sequence has T / B."""
    pages = paged.KVPages.alloc(64, 4, 256, "int8", 64, "cpu")
    f = _C.lib().qvex_paged_attention_workspace_bytes
    for B, T, rows in ((1, 16, 8), (2, 8, 9), (2, 32, 8), (2, 32, 64), (2, 128, 100), (8, 4, 2)):
        got = paged.workspace_bytes(pages, B, T, 16, 4000, max_rows=rows)
        assert got >= f(B, rows, T, 16, 4, 256, 4000, 0) and got >= f(B, max(T // B, 1), T, 16, 4, 256, 4000, 0)


def test_caches_grow_together_or_not_at_all():
    """Layers of one model: pages for all of them, or an error that leaves every cache and the pool as they were."""
    from qvex.model import CacheCounters, KVCache
    counters = CacheCounters(4, "cpu")
    pool, other = (paged.PagePool(40, 2, 128, "int8", 16, "cpu") for _ in range(2))
    dense = KVCache(counters, 3, n_kv=2, head_dim=64, capacity=256, device="cpu")
    caches = [paged.PagedKVCache(other, counters, 0, capacity=1), paged.PagedKVCache(pool, counters, 1, capacity=1), dense,
              paged.PagedKVCache(pool, counters, 2, capacity=1)]
    for c in caches:
        c.offset = 250
    kv = [caches[0], caches[1], caches[3]]
    before = [(list(c.ids), c.table.tolist()) for c in kv], list(pool.holders), list(other.holders)
    with pytest.raises(_C.QvexError, match="free pages"):
        paged.PagedKVCache.grow_all(caches, 7)           # 8 pages left in the pool, 16 and 16 more are needed
    assert before == ([(list(c.ids), c.table.tolist()) for c in kv], list(pool.holders), list(other.holders))
    paged.PagedKVCache.grow_all(caches, 6)               # they fit
    assert before[0] == [(list(c.ids), c.table.tolist()) for c in kv]
    pool.growable = True
    paged.PagedKVCache.grow_all(caches, 7)
    for c, (ids, _) in zip(kv, before[0]):
        assert c.capacity == 512 and c.ids[:16] == ids and c.table[0].tolist() == c.ids and c.offset == 250
    assert dense.capacity == 256
    counters.graph_mode = True
    with pytest.raises(_C.QvexError, match="captured cycle"):
        paged.PagedKVCache.grow_all(caches, 300)


def test_caches_of_a_small_pool_grow_by_what_it_has():
    """Before a captured cycle: by the positions asked for, by less where the pool has less, and an error below `least`."""
    from qvex.model import KVCache
    from qvex.speculative import grow_kv
    pool = paged.PagePool(112, 2, 128, "int8", 16, "cpu")
    caches = [paged.PagedKVCache(pool, capacity=256) for _ in range(2)]
    dense = KVCache(None, 0, n_kv=2, head_dim=64, capacity=256, device="cpu")
    for c in (*caches, dense):
        c.offset = 250
    with pytest.raises(_C.QvexError, match="free pages"):
        grow_kv([*caches, dense], 2048)
    assert [c.capacity for c in (*caches, dense)] == [256, 256, 256]
    assert grow_kv([*caches, dense], 2048, 16)                 # 80 pages: 512 positions for each, then
    assert [c.capacity for c in (*caches, dense)] == [768, 768, 2304]
    assert not grow_kv(caches, 100, 16)
    for c in caches:
        c.offset = 760
    with pytest.raises(_C.QvexError, match="free pages"):
        grow_kv(caches, 2048, 16)                              # 16 pages are left, 32 are needed
    assert [c.capacity for c in caches] == [768, 768] and len(pool.free) == 16
    assert grow_kv(caches[:1], 2048, 16) and [c.capacity for c in caches] == [1024, 768] and not pool.free
