"""The model on paged caches (Qwen35.make_cache(kv=...)): an attention layer against float64 over
what its pages hold, decode() on the captured cycle, growth, shared prefixes, generate()."""

import pytest
import torch

import paged_ref as ref
from qvex import _C, paged
from qvex.engine import generate, prefill
from qvex.model import Config, random_model
from qvex.mtp import random_mtp
from qvex.sampler import Sampler, SamplingParams
from qvex.speculative import decode

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "int8", "fp8"]


@pytest.fixture(scope="module")
def tiny(dev):
    model = random_model(Config.tiny(layers=4, vocab=2048), seed=5, device=dev, max_context=512)
    return model, random_mtp(model, seed=6)


def ids_of(n, vocab, seed=0):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(0, vocab, (1, n), generator=g, dtype=torch.int32)


class _Keep:
    """An o_proj that keeps what it was given."""

    def __call__(self, o):
        self.o = o
        return o


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [[1, 4, 8], [70, 9, 1, 130]])
def test_attention_layer_over_pages(dev, tiny, fmt, rows):
    """Chunks and single rows through Attention on a paged cache, against float64 attention over the
    values that the pages stand for (q from the input stage run again on a pool of its own)."""
    model, _ = tiny
    cfg, layer = model.cfg, next(l.mixer for l in model.layers if not l.linear)
    H, n_kv, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    cache = model.make_cache(max_context=256, kv=fmt)[-1]
    keep, o_proj = _Keep(), layer.o_proj
    layer.o_proj = keep
    try:
        at = 0
        for n in rows:
            g = torch.Generator()
            g.manual_seed(n)
            x = torch.randn((n, cfg.hidden_size), generator=g).to(torch.bfloat16).to(dev)
            proj = layer.qkv_proj(x)
            cache.counters.sync()
            layer(x, cache)
            assert cache.offset == at + n
            pool = ref.Pool(cache.pages.n_pages, n_kv, cache.pages.page, D, fmt)
            pool.k, pool.v = cache.pages.k.cpu(), cache.pages.v.cpu()
            if fmt != "bf16":
                pool.ks, pool.vs = cache.pages.k_scale.cpu(), cache.pages.v_scale.cpu()
            scratch = paged.KVPages.alloc(cache.pages.n_pages, n_kv, D, fmt, cache.pages.page, dev)
            q = paged.attn_qk_rope(scratch, proj, layer.q_norm, layer.k_norm, cache.table,
                                   torch.tensor([at], dtype=torch.int32, device=dev),
                                   paged.rope_freqs(cfg.rotary_dim, cfg.rope_theta, dev), cfg.rms_norm_eps)
            gate = proj.cpu()[:, :2 * H * D].reshape(n, H, 2 * D)[..., D:]
            want, tol = ref.attention(pool, q.cpu(), cache.table.tolist(), [at], None, gate, terms=2 if n <= 8 else 1)
            assert bool(((keep.o.cpu().double().view(n, H, D) - want).abs() <= tol).all())
            at += n
    finally:
        layer.o_proj = o_proj
    k = cache.keys()
    assert k.shape == (n_kv, cache.capacity, D) and bool((k[:, at:] == 0).all()) and bool((k[:, :at] != 0).any())


def run(model, mtp, ids, kv, n, graph=True, k=3, temperature=0.0, use_mtp=True, cap=None):
    cache = model.make_cache(max_context=cap, kv=kv)
    mc = mtp.make_cache(max_context=cap, kv=kv)
    logits, last = prefill(model, ids, cache, mtp, mc)
    smp = Sampler(SamplingParams(temperature=temperature, top_k=20 if temperature else 0,
                                 top_p=0.8 if temperature else 1.0, seed=3), model.cfg.vocab_size)
    st: dict = {}
    gen = decode(model, smp, cache, logits[0, -1], last, mtp, mc, lambda: use_mtp, st, k=k, graph=graph)
    out = [next(gen) for _ in range(n)]
    gen.close()
    return out, st, cache


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_is_the_same_captured_eager_and_plain(tiny, fmt):
    """On pages as on dense caches: the captured cycle emits the eager one's tokens (sampled too), and greedy
    speculation emits plain greedy decoding's."""
    model, mtp = tiny
    ids = ids_of(77, model.cfg.vocab_size)
    a, st, _ = run(model, mtp, ids, fmt, 24)
    assert st["graph_cycles"] > 0
    assert a == run(model, mtp, ids, fmt, 24, graph=False)[0]
    assert a == run(model, mtp, ids, fmt, 24, use_mtp=False)[0]
    s = run(model, mtp, ids, fmt, 24, temperature=0.9)[0]
    assert s == run(model, mtp, ids, fmt, 24, graph=False, temperature=0.9)[0]


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_past_the_capacity_grows(tiny, fmt):
    """A prompt that ends 3 positions before the capacity: the caches grow, in the captured path too."""
    model, mtp = tiny
    ids = ids_of(253, model.cfg.vocab_size, seed=1)
    a, _, cache = run(model, mtp, ids, fmt, 20, cap=256)
    assert cache[-1].capacity > 256
    assert a == run(model, mtp, ids, fmt, 20, cap=1024)[0]
    assert a == run(model, mtp, ids, fmt, 20, cap=256, graph=False)[0]


def test_two_branches_of_a_shared_prefix(dev, tiny):
    """Sequences that share a prefix's pages go on as if each had its own, also after a rollback into it."""
    model, _ = tiny
    V = model.cfg.vocab_size
    pool = paged.PagePool(200, model.cfg.num_key_value_heads, model.cfg.head_dim, "int8", 16, dev)

    def more(cache, ids):
        return model(ids, cache, last_only=False).clone()

    def fresh(*parts):
        cache = model.make_cache(max_context=256, kv="int8")
        out = None
        for p in parts:
            out = more(cache, p)
        return out

    prefix, x, y = ids_of(61, V, 2), ids_of(7, V, 3), ids_of(5, V, 4)
    a = model.make_cache(max_context=256, kv=pool)
    more(a, prefix)
    used = 200 - len(pool.free)
    b = a.clone()
    assert 200 - len(pool.free) < 2 * used        # the whole pages of the prefix are not copied
    assert torch.equal(more(b, y), fresh(prefix, y)) and torch.equal(more(a, x), fresh(prefix, x))
    z = ids_of(3, V, 5)
    assert torch.equal(more(b, z), fresh(prefix, y, z)) and torch.equal(more(a, z), fresh(prefix, x, z))
    del a, b
    assert len(pool.free) == 200


def test_rollback_into_a_shared_page(dev, tiny):
    """KV pages only (a verify of rejected drafts after a clone): the twin's keys stay."""
    model, _ = tiny
    cfg = model.cfg
    pool = paged.PagePool(40, cfg.num_key_value_heads, cfg.head_dim, "int8", 16, dev)
    a = paged.PagedKVCache(pool, capacity=64)
    g = torch.Generator()
    g.manual_seed(9)
    kv = torch.randn((40, cfg.num_key_value_heads, cfg.head_dim), generator=g).to(torch.bfloat16).to(dev)

    def put(c, rows):
        c.counters.sync()
        paged.kv_append(c.pages, rows, rows, c.table, c.pos)
        c.offset += rows.shape[0]

    put(a, kv)
    b = a.clone()
    kept = b.keys()[:, :40].clone()
    a.rollback(20)
    put(a, -kv[:20])
    assert torch.equal(b.keys()[:, :40], kept) and torch.equal(b.values()[:, :40], kept)
    k = a.keys()
    assert torch.equal(k[:, :20], kept[:, :20]) and torch.equal(k[:, 20:40], -kept[:, :20])


def test_generate_on_pages(tiny):
    model, mtp = tiny
    params = SamplingParams(temperature=0.0, top_k=0, top_p=1.0, max_tokens=20)
    ids = ids_of(40, model.cfg.vocab_size, 6)
    for fmt in FORMATS:
        on = generate(model, ids, params, mtp, "on", kv=fmt)
        off = generate(model, ids, params, mtp, "off", kv=fmt)
        assert on.tokens == off.tokens and len(on.tokens) == 20 and on.stats["mtp_cycles"] > 0
    pool = paged.PagePool(64, model.cfg.num_key_value_heads, model.cfg.head_dim, "int8", 64, model.norm.device)
    assert generate(model, ids, params, mtp, "on", kv=pool).tokens == generate(model, ids, params, mtp, "on", kv="int8").tokens
    assert len(pool.free) == 64
    with pytest.raises(_C.QvexError, match="unknown KV format"):
        generate(model, ids, params, mtp, "on", kv="int4")
    with pytest.raises(_C.QvexError, match="page pool holds"):
        model.make_cache(kv=paged.PagePool(4, 1, 128, "int8", 64, model.norm.device))


def test_bf16_pages_and_dense_caches_agree(tiny):
    """The same prompt, chunk and steps: logits within two bf16 steps of the largest."""
    model, _ = tiny
    V = model.cfg.vocab_size
    outs = []
    for kv in (None, "bf16"):
        cache = model.make_cache(max_context=512, kv=kv)
        outs.append([model(ids_of(n, V, n), cache, last_only=False).float() for n in (130, 40, 4, 1)])
    for a, b in zip(*outs):
        assert float((a - b).abs().max()) <= 2 * 2.0 ** -7 * float(a.abs().max())


@pytest.mark.parametrize("fmt", [None, *FORMATS])
def test_one_token_prompt_on_a_fresh_head(dev, fmt):
    """The first call of the MTP head's attention is inside the capture of the cycle (a prompt of one token leaves it no pair)."""
    model = random_model(Config.tiny(layers=4, vocab=2048), seed=7, device=dev, max_context=256)
    params = SamplingParams(temperature=0.0, top_k=0, top_p=1.0, max_tokens=12)
    on = generate(model, [17], params, random_mtp(model, seed=8), "on", kv=fmt)
    assert on.stats["mtp_graph_cycles"] == on.stats["mtp_cycles"] > 0
    assert on.tokens == generate(model, [17], params, None, "off", kv=fmt).tokens and len(on.tokens) == 12


def test_generate_takes_what_it_needs_of_a_pool(dev, tiny):
    """Pages for the prompt and max_tokens, not for the model's max_context: two sequences of one fixed pool at a
    time (the second held by a cache), and a call that needs more raises with the pool as it was."""
    model = random_model(Config.tiny(layers=4, vocab=2048), seed=5, device=dev, max_context=4096)
    mtp = random_mtp(model, seed=6)
    cfg = model.cfg
    params = SamplingParams(temperature=0.0, top_k=0, top_p=1.0, max_tokens=20)
    ids = ids_of(40, cfg.vocab_size, 6)
    pool = paged.PagePool(12, cfg.num_key_value_heads, cfg.head_dim, "int8", 64, dev)
    other = model.make_cache(max_context=200, kv=pool)              # 4 pages; the call: 4 for the layer, 4 for the head
    got = generate(model, ids, params, mtp, "on", kv=pool)
    assert got.tokens == generate(model, ids, params, mtp, "on", kv="int8").tokens and got.stats["mtp_graph_cycles"] > 0
    assert got.tokens == generate(model, ids, params, mtp, "on", kv=pool, max_tokens=20).tokens
    assert len(pool.free) == 8
    with pytest.raises(_C.QvexError, match="free pages of 12"):
        generate(model, ids, params, mtp, "on", kv=pool, max_tokens=300)
    del other
    assert len(pool.free) == 12


@pytest.mark.parametrize("n", [7, 40, 600])
def test_a_call_without_pages_leaves_every_layer_as_it_was(dev, n):
    """A pool that runs out at the second attention layer: the first one, and the recurrent ones, have not moved, and
    the call goes through once there are pages."""
    model = random_model(Config.tiny(layers=8, vocab=2048), seed=9, device=dev, max_context=256)
    cfg = model.cfg
    page = 64
    need = -(-(250 + n) // 256) * 256 // page - 4                   # more pages of each of the two layers
    pool = paged.PagePool(8 + need, cfg.num_key_value_heads, cfg.head_dim, "int8", page, dev)
    prompt, more = ids_of(250, cfg.vocab_size, 1), ids_of(n, cfg.vocab_size, 2)
    cache = model.make_cache(max_context=256, kv=pool)
    model(prompt, cache)
    with pytest.raises(_C.QvexError, match="free pages"):
        model(more, cache)
    assert cache.counters.host.tolist() == [250] * 8
    pool.growable = True
    got = model(more, cache, last_only=False)
    other = model.make_cache(max_context=1024, kv="int8")
    model(prompt, other)
    assert torch.equal(got, model(more, other, last_only=False))


@pytest.mark.parametrize("graph", [True, False])
def test_decode_grows_by_what_a_small_pool_has(dev, tiny, graph):
    """A fixed pool that two caches outgrow by 256 positions each: the captured cycle's larger steps are not taken, its
    tokens are those of a pool of its own; past the last page the error leaves the caches with their keys."""
    model, mtp = tiny
    cfg = model.cfg
    ids = ids_of(240, cfg.vocab_size, 7)
    want, _, _ = run(model, mtp, ids, "int8", 60, cap=1024)
    pool = paged.PagePool(16, cfg.num_key_value_heads, cfg.head_dim, "int8", 64, dev)
    got, st, cache = run(model, mtp, ids, pool, 60, graph=graph, cap=256)
    assert got == want and cache[-1].capacity == 512 and not cache.counters.graph_mode
    assert not graph or st["graph_cycles"] > 0
    with pytest.raises(_C.QvexError, match="free pages"):
        run(model, mtp, ids, pool, 300, graph=graph, cap=256)
