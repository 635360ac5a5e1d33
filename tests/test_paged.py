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
          dict(ws=None), dict(ws=8), dict(ws_bytes=16)]


@pytest.mark.parametrize("bad", COMMON + [dict(prefix_len=-1), dict(prefix_pages=None), dict(max_len=-1)], ids=str)
def test_shared_prefix_attention_refuses(bad):
    assert _shared(**bad) == _abi.MQ_ERR_ARG


@pytest.mark.parametrize("bad", COMMON + [dict(chosen=None), dict(top=0), dict(top=8193)], ids=str)
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
