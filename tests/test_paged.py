"""CPU tests of the paged K/V cache: what the C entries and the Python functions refuse, before
any launch (no kernel runs here)."""

import ctypes

import pytest
import torch

from megaqwen_amd import _abi, paged

BF = torch.bfloat16


def _pool(**over):
    a = dict(k=16, v=16, bounds=16, num_layers=1, num_pages=8, num_kv_heads=2, page_size=16, head_dim=64, dtype=_abi.MQ_BF16)
    a.update(over)
    return _abi.MqPagePool(*a.values())


BAD_POOLS = [dict(k=None), dict(v=None), dict(k=8), dict(v=24), dict(bounds=8), dict(num_pages=0), dict(num_kv_heads=0),
             dict(num_layers=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(head_dim=96), dict(dtype=2),
             dict(dtype=-1)]


def _ints(*x):
    return (ctypes.c_int * len(x))(*x)


def _copy(pool=None, src=(0,), dst=(1,), n=1):
    return _abi.lib().mq_pages_copy(pool or _pool(), _ints(*src), _ints(*dst), n, None)


def _load(pool=None, pages=(0, 1), length=20, k=16, v=16, max_seq=32, entry="mq_pages_load"):
    return getattr(_abi.lib(), entry)(pool or _pool(), _ints(*pages), length, k, v, max_seq, None)


def _append(pool=None, **over):
    a = dict(k=16, v=16, k_sb=128, k_sh=64, v_sb=128, v_sh=64, tables=16, t_sb=4, width=4, lens=16, batch=3)
    a.update(over)
    return _abi.lib().mq_pages_append(pool or _pool(), *a.values(), None)


def _shared(pool=None, **over):
    a = dict(q=16, q_sb=256, q_sh=64, out=16, o_sb=256, o_sh=64, heads=4, batch=3, prefix_pages=16, prefix_len=20, tables=16, t_sb=4,
             width=4, lens=16, max_len=64, scale=0.1, ws=16, ws_bytes=1 << 30)
    a.update(over)
    return _abi.lib().mq_shared_prefix_attention(pool or _pool(), *a.values(), None)


def _sparse(pool=None, **over):
    a = dict(q=16, q_sb=256, q_sh=64, out=16, o_sb=256, o_sh=64, chosen=16, heads=4, batch=3, tables=16, t_sb=4, width=4, lens=16,
             top=2, scale=0.1, ws=16, ws_bytes=1 << 30)
    a.update(over)
    return _abi.lib().mq_sparse_attention(pool or _pool(), *a.values(), None)


@pytest.mark.parametrize("bad", BAD_POOLS, ids=str)
def test_entries_refuse_a_bad_pool(bad):
    for call in (_copy, _load, _append, _shared, _sparse):
        assert call(_pool(**bad)) == _abi.MQ_ERR_ARG
    assert _load(_pool(**bad), entry="mq_pages_store") == _abi.MQ_ERR_ARG


@pytest.mark.parametrize("bad", [dict(src=(-1,)), dict(src=(8,)), dict(dst=(8,)), dict(dst=(-2,)), dict(n=-1)], ids=str)
def test_copy_refuses(bad):
    assert _copy(**bad) == _abi.MQ_ERR_ARG


@pytest.mark.parametrize("entry", ["mq_pages_load", "mq_pages_store"])
@pytest.mark.parametrize("bad", [dict(pages=(0, 8)), dict(pages=(-1, 0)), dict(length=0), dict(length=33), dict(k=None), dict(v=None),
                                 dict(k=8), dict(max_seq=19)], ids=str)
def test_load_and_store_refuse(entry, bad):
    assert _load(**{"pages": (0, 1, 2), **bad}, entry=entry) == _abi.MQ_ERR_ARG


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=8), dict(k_sb=129), dict(v_sh=68), dict(tables=None), dict(lens=None),
                                 dict(width=0), dict(width=8193), dict(t_sb=-4), dict(batch=0), dict(batch=65536)], ids=str)
def test_append_refuses(bad):
    assert _append(**bad) == _abi.MQ_ERR_ARG


COMMON = [dict(q=None), dict(q=8), dict(out=None), dict(out=24), dict(q_sb=4), dict(q_sh=65), dict(o_sb=1), dict(o_sh=4), dict(heads=0),
          dict(heads=1), dict(heads=3), dict(batch=0), dict(batch=65536), dict(tables=None), dict(lens=None), dict(width=0),
          dict(width=8193), dict(t_sb=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
          dict(scale=-0.0)]


@pytest.mark.parametrize("bad", COMMON + [dict(prefix_len=-1), dict(prefix_len=2 ** 30 + 1), dict(prefix_pages=None), dict(max_len=-1), dict(max_len=2 ** 31 - 1), dict(prefix_len=2000, ws_bytes=16),
                                          dict(prefix_len=2000, ws=None), dict(prefix_len=2000, ws=8)], ids=str)
def test_shared_prefix_attention_refuses(bad):
    assert _shared(**bad) == _abi.MQ_ERR_ARG


@pytest.mark.parametrize("bad", COMMON + [dict(chosen=None), dict(top=0), dict(top=8193), dict(ws_bytes=16), dict(ws=None), dict(ws=8)], ids=str)
def test_sparse_attention_refuses(bad):
    assert _sparse(**bad) == _abi.MQ_ERR_ARG
    assert _sparse(_pool(bounds=None)) == _abi.MQ_ERR_ARG


def test_workspace_query():
    L, n = _abi.lib(), ctypes.c_size_t()
    for bad in ((_pool(), 3, 1, 0, 16, 0), (_pool(), 4, 0, 0, 16, 0), (_pool(), 4, 1, -1, 16, 0), (_pool(), 4, 1, 0, -1, 0),
                (_pool(), 4, 1, 0, 16, -1), (_pool(num_kv_heads=0), 4, 1, 0, 16, 0)):
        assert L.mq_attention_workspace(*bad, n) == _abi.MQ_ERR_ARG
    got = []
    for batch in (1, 4, 64):
        assert L.mq_attention_workspace(_pool(), 4, batch, 1000, 500, 0, n) == _abi.MQ_OK
        got.append(n.value)
    assert 0 < got[0] and got[2] < 1 << 28
    assert L.mq_attention_workspace(_pool(), 4, 4, 0, 500, 7, n) == _abi.MQ_OK and n.value >= 4 * 2 * 7 * 4


# ---------------------------------------------------------------- the Python functions

K = torch.zeros(2, 8, 2, 16, 64, dtype=BF)
B = torch.zeros(2, 8, 2, 2, 64, dtype=BF)
CACHE = torch.zeros(2, 2, 40, 64, dtype=BF)
ROWS = torch.zeros(3, 2, 64, dtype=BF)
Q = torch.zeros(3, 4, 64, dtype=BF)
T, LENS = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)


def _refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


@pytest.mark.parametrize("k,v,match", [
    (K[0], K[0], "5 dimensions"), (K.float(), K.float(), "bfloat16"), (K, K[:1], "v_pages"), (K, K.half(), "v_pages"),
    (K[:, :, :, :9], K[:, :, :, :9], "page size 9"), (K[..., :32], K[..., :32], "head dim 32"), (K[:, ::2], K[:, ::2], "contiguous"),
    (K[:, :0], K[:, :0], "size of zero"), (None, K, "k_pages")])
def test_pool_refusals(k, v, match):
    _refused(match, paged.copy_pages, k, v, [0], [1])
    _refused(match, paged.load_pages, CACHE, CACHE, k, v, [0], 5)
    _refused(match, paged.store_pages, k, v, [0], 5, CACHE, CACHE)


def test_copy_refusals():
    for src, dst, match in (([0, 1], [2], "one length"), ([0, 1], [2, 2], "twice"), ([0, 1], [1, 2], "copied from"), ([3], [3], "copied"),
                            ([-1], [2], "src"), ([8], [2], "src"), ([1], [8], "dst")):
        _refused(match, paged.copy_pages, K, K, src, dst)
    _refused("bounds", paged.copy_pages, K, K, [0], [1], bounds=B[:, :4])
    _refused("bounds", paged.copy_pages, K, K, [0], [1], bounds=B.half())
    _refused("on the GPU", paged.copy_pages, K, K, [0], [1], bounds=B)


def test_load_and_store_refusals():
    for pages, n, match in (([0], 17, "pages"), ([0, 1], 16, "pages"), ([0, 0], 20, "twice"), ([0, 8], 20, "pages"), ([0, 1, 2], 41, "exceeds"),
                            ([], -1, "pages")):
        _refused(match, paged.load_pages, CACHE, CACHE, K, K, pages, n)
        _refused(match, paged.store_pages, K, K, pages, n, CACHE, CACHE)
    _refused("k_cache", paged.load_pages, CACHE[0], CACHE, K, K, [0], 5)
    _refused("k_cache", paged.load_pages, CACHE[:1], CACHE[:1], K, K, [0], 5)
    _refused("v_cache", paged.load_pages, CACHE, CACHE[:, :, :30], K, K, [0], 5)
    _refused("contiguous", paged.load_pages, CACHE[:, :, ::2], CACHE[:, :, ::2], K, K, [0], 5)
    _refused("k_cache", paged.load_pages, CACHE.half(), CACHE, K, K, [0], 5)
    _refused("on the GPU", paged.load_pages, CACHE, CACHE, K, K, [0], 5)
    _refused("on the GPU", paged.store_pages, K, K, [0], 5, CACHE, CACHE)
    paged.load_pages(CACHE, CACHE, K, K, [], 0)  # nothing to do


def test_append_refusals():
    k = K[0]
    bad = [((ROWS[0], ROWS, k, k, T, LENS), "k:"), ((ROWS, ROWS[:2], k, k, T, LENS), "v:"), ((ROWS.half(), ROWS, k, k, T, LENS), "k:"),
           ((torch.zeros(3, 2, 128, dtype=BF)[..., ::2], ROWS, k, k, T, LENS), "strides"),
           ((torch.zeros(3, 2, 66, dtype=BF)[..., :64], ROWS, k, k, T, LENS), "strides"),
           ((torch.zeros(3 * 128 + 1, dtype=BF)[1:].view(3, 2, 64), ROWS, k, k, T, LENS), "16 bytes"),
           ((ROWS, ROWS, k, k, T[:2], LENS), "tables"), ((ROWS, ROWS, k, k, T.long(), LENS), "tables"),
           ((ROWS, ROWS, k, k, T[:, :0], LENS), "tables"), ((ROWS, ROWS, k, k, torch.zeros(3, 8, dtype=torch.int32)[:, ::2], LENS), "rows"),
           ((ROWS, ROWS, k, k, T, LENS[:2]), "lens"), ((ROWS, ROWS, k, k, T, LENS.long()), "lens"), ((ROWS, ROWS, K, K, T, LENS), "k_pages"),
           ((ROWS, ROWS, k, k, T, LENS), "on the GPU")]
    for args, match in bad:
        _refused(match, paged.append_rows, *args)


def test_attention_refusals():
    k, b = K[0], B[0]
    pre = torch.zeros(2, dtype=torch.int32)
    shared, sparse = paged.shared_prefix_attention, paged.sparse_attention
    for q, match in ((Q[0], "q:"), (Q[:, :3], "q:"), (Q.float(), "q:"), (Q[..., :32], "q:"), (torch.zeros(3, 4, 68, dtype=BF)[..., :64], "strides")):
        _refused(match, shared, q, k, k, pre, 20, T, LENS)
        _refused(match, sparse, q, k, k, b, T, LENS, 2)
    for scale in (0.0, -0.5, float("nan"), float("inf")):
        _refused("scale", shared, Q, k, k, pre, 20, T, LENS, scale=scale)
        _refused("scale", sparse, Q, k, k, b, T, LENS, 2, scale=scale)
    for out in (Q[:2], Q.half(), torch.zeros(1, 4, 64, dtype=BF).expand(3, 4, 64)):
        _refused("out", shared, Q, k, k, pre, 20, T, LENS, out=out)
        _refused("out", sparse, Q, k, k, b, T, LENS, 2, out=out)
    _refused("prefix_len", shared, Q, k, k, pre, -1, T, LENS)
    _refused("prefix_pages", shared, Q, k, k, pre, 33, T, LENS)
    _refused("prefix_pages", shared, Q, k, k, pre.long(), 20, T, LENS)
    _refused("prefix_pages", shared, Q, k, k, None, 20, T, LENS)
    _refused("max_len", shared, Q, k, k, pre, 20, T, LENS, max_len=0)
    _refused("tables", shared, Q, k, k, pre, 20, T[:2], LENS)
    _refused("lens", sparse, Q, k, k, b, T, LENS[:1], 2)
    _refused("top_pages", sparse, Q, k, k, b, T, LENS, 0)
    _refused("top_pages", sparse, Q, k, k, b, T, LENS, 8193)
    _refused("bounds", sparse, Q, k, k, None, T, LENS, 2)
    _refused("bounds", sparse, Q, k, k, b[:4], T, LENS, 2)
    _refused("on the GPU", shared, Q, k, k, pre, 20, T, LENS)
    _refused("on the GPU", sparse, Q, k, k, b, T, LENS, 2)


def test_outputs_that_overlap_are_refused():
    pre, k, b = torch.zeros(2, dtype=torch.int32), K[0], B[0]
    flat = torch.zeros(4096, dtype=BF)
    for strides, ok in (((256, 64, 1), True), ((64, 192, 1), True), ((512, 128, 1), True), ((256, 56, 1), False), ((128, 64, 1), False),
                        ((8, 64, 1), False), ((64, 64, 1), False), ((64, 128, 1), False)):
        out = flat.as_strided((3, 4, 64), strides)
        _refused("on the GPU" if ok else "overlap", paged.shared_prefix_attention, Q, k, k, pre, 20, T, LENS, out=out)
        _refused("on the GPU" if ok else "overlap", paged.sparse_attention, Q, k, k, b, T, LENS, 2, out=out)
    one = flat.as_strided((1, 4, 64), (8, 64, 1))  # (a stride over one element does not matter)
    _refused("on the GPU", paged.shared_prefix_attention, Q[:1], k, k, pre, 20, T[:1], LENS[:1], out=one)


def test_entries_refuse_what_passes_their_limits():
    L, n = _abi.lib(), ctypes.c_size_t()
    ids = (ctypes.c_int * 1)(0)
    for entry in (L.mq_pages_load, L.mq_pages_store):
        assert entry(_pool(), ids, 2**31 - 1, 16, 16, 2**31 - 1, None) == _abi.MQ_ERR_ARG
    for bad in ((_pool(), 16386, 1, 0, 16, 0), (_pool(), 4, 65536, 0, 16, 0), (_pool(), 4, 1, 0, 16, 8193)):
        assert L.mq_attention_workspace(*bad, n) == _abi.MQ_ERR_ARG
    for bad in (dict(k=24), dict(v=24), dict(bounds=24)):
        assert _batch(_model_pool(**bad)) == _abi.MQ_ERR_ARG


# ---------------------------------------------------------------- the batched decode step

def _layers(n=2, **over):
    arr = (_abi.LDGLayerWeights * n)()
    for i in range(n):
        for name in _abi.LAYER_FIELDS:
            setattr(arr[i], name, over.get(name, 16))
    return arr


def _batch(pool=None, made=None, **over):
    made = _layers() if made is None else made
    a = dict(ids=16, out=16, logits=None, batch=3, embed=16, layers=ctypes.addressof(made), norm=16, lm=16, cos=16, sin=16,
             num_positions=100, pool=pool or _model_pool(), prefix_pages=16, prefix_len=64, tables=16, t_sb=4, width=4, lens=16,
             max_len=64, top=0, scale=0.1, ws=256, ws_bytes=1 << 40)
    a.update(over)
    return _abi.lib().mq_decode_batch(*a.values(), None)


def _model_pool(**over):
    return _pool(**{**dict(num_layers=2, num_kv_heads=8, page_size=64, head_dim=128), **over})


@pytest.mark.parametrize("bad", [
    dict(ids=None), dict(out=None), dict(batch=0), dict(batch=1025), dict(embed=None), dict(layers=None), dict(norm=None), dict(lm=None),
    dict(cos=None), dict(sin=None), dict(num_positions=64), dict(prefix_pages=None), dict(prefix_len=-1), dict(tables=None), dict(t_sb=-1),
    dict(width=0), dict(width=8193), dict(lens=None), dict(max_len=0), dict(top=-1), dict(top=4), dict(scale=0.0), dict(scale=float("nan")),
    dict(ws=None), dict(ws=128), dict(ws_bytes=1000), dict(pool=_model_pool(num_kv_heads=4)), dict(pool=_model_pool(head_dim=64)),
    dict(pool=_model_pool(dtype=_abi.MQ_FP16)), dict(pool=_model_pool(num_layers=33)), dict(pool=_model_pool(page_size=24)),
    dict(pool=_model_pool(k=None)), dict(pool=_model_pool(num_pages=0)), dict(pool=_model_pool(bounds=None), top=4, prefix_len=0)], ids=str)
def test_decode_batch_refuses(bad):
    assert _batch(**bad) == _abi.MQ_ERR_ARG


def test_decode_batch_refuses_a_missing_weight():
    assert _batch(made=_layers(down_proj_weight=None)) == _abi.MQ_ERR_ARG


def test_decode_batch_workspace_query():
    L, n = _abi.lib(), ctypes.c_size_t()
    for bad in ((_model_pool(num_kv_heads=2), 3, 0, 64, 0, 4), (_model_pool(), 0, 0, 64, 0, 4), (_model_pool(), 3, 64, 64, 4, 4),
                (_model_pool(), 3, 0, 0, 0, 4), (_model_pool(), 3, 0, 64, 0, 0)):
        assert L.mq_decode_batch_workspace(*bad, n) == _abi.MQ_ERR_ARG
    assert L.mq_decode_batch_workspace(_model_pool(), 3, 640, 64, 0, 4, n) == _abi.MQ_OK
    assert n.value >= 3 * 151936 * 2


# ---------------------------------------------------------------- the books

@pytest.fixture
def cpu_pages(monkeypatch):
    """The page moves on the CPU, so that the books can be checked without a GPU."""
    def copy(k, v, src, dst, bounds=None):
        assert len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst)
        for t in (k, v):
            t[:, dst] = t[:, src].clone()

    def load(kc, vc, k, v, pages, length, bounds=None):
        for t, c in ((k, kc), (v, vc)):
            for i in range(length):
                t[:, pages[i // t.shape[3]], :, i % t.shape[3]] = c[:, :, i]

    def store(k, v, pages, length, kc, vc):
        for t, c in ((k, kc), (v, vc)):
            for i in range(length):
                c[:, :, i] = t[:, pages[i // t.shape[3]], :, i % t.shape[3]]

    monkeypatch.setattr(paged, "copy_pages", copy)
    monkeypatch.setattr(paged, "load_pages", load)
    monkeypatch.setattr(paged, "store_pages", store)


def _cache(num_pages=40, page_size=16):
    return paged.PagedKVCache(num_pages, 1, 1, 64, page_size, torch.bfloat16, "cpu")


def _grow(cache, seqs, values):
    """What append_rows does to position length(seq)."""
    cache.reserve(seqs)
    for s, x in zip(seqs, values):
        n, p = cache.length(s), cache.page_size
        cache.k_pages[0, cache.pages(s)[n // p], 0, n % p, 0] = x
    cache.extend(seqs)


def _rows(cache, seq):
    kc, vc = torch.zeros(1, 1, 400, 64, dtype=BF), torch.zeros(1, 1, 400, 64, dtype=BF)
    n = cache.store(seq, kc, vc)
    assert n == cache.length(seq)
    return kc[0, 0, :n, 0].tolist()


def _check_books(cache):
    users = [0] * cache.num_pages
    for pages, n in cache._seqs.values():
        assert len(set(pages)) == len(pages) and n <= len(pages) * cache.page_size
        for p in pages:
            users[p] += 1
    assert users == cache._users
    assert sorted(cache._free) == [p for p, u in enumerate(users) if u == 0]


@pytest.mark.parametrize("seed", range(6))
def test_cache_against_plain_lists(cpu_pages, seed):
    """Random forks, appends, frees and compactions; every sequence's rows are those of a list of its own."""
    import random

    rng = random.Random(seed)
    cache, plain = _cache(), {}
    root = cache.new()
    plain[root] = []
    for step in range(300):
        op = rng.choice(["append", "append", "append", "append", "fork", "free", "compact"])
        live = list(plain)
        if op == "append" and live:
            seqs = rng.sample(live, rng.randint(1, len(live)))
            values = [float(rng.randint(-128, 128)) for _ in seqs]
            try:
                _grow(cache, seqs, values)
            except _abi.MegakernelError:
                _check_books(cache)  # (nothing has changed)
                victim = rng.choice(live)
                cache.free(victim)
                del plain[victim]
            else:
                for s, x in zip(seqs, values):
                    plain[s].append(x)
        elif op == "fork" and live and len(live) < 9:
            s, n = rng.choice(live), rng.randint(0, 3)
            for t in cache.fork(s, n):
                plain[t] = list(plain[s])
        elif op == "free" and len(live) > 3:
            s = rng.choice(live)
            cache.free(s)
            del plain[s]
        elif op == "compact":
            used = cache.compact()
            assert used == cache.num_pages - cache.free_pages() and sorted(cache._free) == list(range(used, cache.num_pages))
        _check_books(cache)
        for s, rows in plain.items():
            assert _rows(cache, s) == rows
    for s in list(plain):
        cache.free(s)
    assert cache.free_pages() == cache.num_pages


def test_fork_copies_a_page_only_when_it_is_written(cpu_pages):
    cache = _cache()
    kc = torch.arange(40, dtype=torch.float32).view(1, 1, 40, 1).expand(1, 1, 40, 64).to(BF).contiguous()
    a = cache.new()
    cache.load(a, kc, kc, 20)  # two pages, the second with 4 rows
    assert cache.pages(a) == [0, 1] and cache.free_pages() == 38
    b, c = cache.fork(a, 2)
    assert cache.pages(b) == cache.pages(c) == [0, 1] and cache.free_pages() == 38
    assert cache.shared_pages([a, b, c]) == 1  # (the full one)
    _grow(cache, [a, b, c], [100.0, 101.0, 102.0])
    # two of the three copied their last page, the last one kept it; the first stays shared
    assert sorted(cache.pages(s)[1] for s in (a, b, c)) == [1, 2, 3] and all(cache.pages(s)[0] == 0 for s in (a, b, c))
    for s, x in ((a, 100.0), (b, 101.0), (c, 102.0)):
        assert _rows(cache, s) == [float(i) for i in range(20)] + [x]
    cache.free(a)
    cache.free(b)
    assert _rows(cache, c)[-1] == 102.0 and cache.free_pages() == 38


def test_a_fork_leaves_reserved_pages_behind(cpu_pages):
    """Pages that hold no row yet are not shared: two sequences that go on from there write to pages of their own."""
    cache = _cache()
    a = cache.new()
    for i in range(16):
        _grow(cache, [a], [float(i)])
    cache.reserve([a], 20)  # pages for positions 16 .. 35
    assert len(cache.pages(a)) == 3
    b = cache.fork(a)[0]
    assert cache.pages(b) == cache.pages(a)[:1]
    _check_books(cache)
    _grow(cache, [a, b], [50.0, 60.0])
    assert cache.pages(a)[1] != cache.pages(b)[1]
    assert _rows(cache, a)[-1] == 50.0 and _rows(cache, b)[-1] == 60.0


def test_every_change_changes_the_version(cpu_pages):
    cache = _cache()
    seen = [cache.version]

    def changed():
        seen.append(cache.version)
        return seen[-1] != seen[-2]

    a = cache.new()
    cache.reserve([a], 3)
    assert changed()
    cache.extend([a], 3)
    assert changed()
    b = cache.fork(a)[0]
    cache.reserve([a], 1)
    assert changed()  # (a page of its own)
    cache.free(a)
    assert changed()
    cache.compact()
    kc = torch.zeros(1, 1, 40, 64, dtype=BF)
    cache.load(cache.new(), kc, kc, 7)
    assert changed() and cache.length(b) == 3


def test_a_full_shared_page_is_not_copied(cpu_pages):
    cache = _cache()
    a = cache.new()
    for i in range(32):
        _grow(cache, [a], [float(i)])
    assert cache.pages(a) == [0, 1]
    b = cache.fork(a)[0]
    _grow(cache, [a, b], [1.0, 2.0])
    assert cache.pages(a)[:2] == cache.pages(b)[:2] == [0, 1] and cache.pages(a)[2] != cache.pages(b)[2]
    assert cache.shared_pages([a, b]) == 2 and cache.shared_pages([a]) == 2


def test_tables_of_a_batch(cpu_pages):
    cache = _cache()
    a = cache.new()
    for i in range(35):
        _grow(cache, [a], [float(i)])
    b = cache.fork(a)[0]
    _grow(cache, [b], [1.0])
    for _ in range(14):
        _grow(cache, [b], [1.0])
    tables, lens = cache.tables([a, b], first=2)
    assert lens.tolist() == [3, 18] and tables.shape == (2, 2) and tables.dtype == torch.int32
    assert tables[0].tolist() == [cache.pages(a)[2], -1] and tables[1].tolist() == cache.pages(b)[2:]
    whole, lens = cache.tables([a])
    assert lens.tolist() == [35] and whole[0].tolist() == cache.pages(a)
    empty, lens = cache.tables([cache.new()])
    assert lens.tolist() == [0] and empty.tolist() == [[-1]]


def test_cache_refusals(cpu_pages):
    for bad in (dict(num_pages=0), dict(num_pages=4, page_size=24), dict(num_pages=4, head_dim=80), dict(num_pages=4, dtype=torch.float32),
                dict(num_pages=4, num_layers=0)):
        with pytest.raises(ValueError):
            paged.PagedKVCache(device="cpu", **bad)
    cache = _cache(num_pages=2)
    a = cache.new()
    for call in (lambda: cache.free(99), lambda: cache.fork(99), lambda: cache.fork(a, -1), lambda: cache.reserve([a, a]),
                 lambda: cache.reserve([a], -1), lambda: cache.extend([a], 1), lambda: cache.length(99), lambda: cache.tables([]),
                 lambda: cache.load(a, CACHE, CACHE, -1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_abi.MegakernelError, match="exhausted"):
        cache.reserve([a], 33)
    assert cache.pages(a) == [] and cache.free_pages() == 2
    kc = torch.zeros(1, 1, 40, 64, dtype=BF)
    with pytest.raises(_abi.MegakernelError, match="exhausted"):
        cache.load(a, kc, kc, 33)
    cache.load(a, kc, kc, 32)
    with pytest.raises(ValueError, match="has rows"):
        cache.load(a, kc, kc, 1)
    cache.free(a)
    with pytest.raises(ValueError):
        cache.free(a)
    assert cache.free_pages() == 2


def test_a_failed_load_gives_its_pages_back():
    cache = _cache(num_pages=4)  # (the real load_pages, which refuses CPU tensors)
    a = cache.new()
    kc = torch.zeros(1, 1, 40, 64, dtype=BF)
    with pytest.raises(ValueError, match="on the GPU"):
        cache.load(a, kc, kc, 20)
    assert cache.free_pages() == 4 and cache.pages(a) == [] and cache.length(a) == 0
