"""GPU tests of the operators on a paged K/V cache (megaqwen_amd.paged) against plain
implementations in 64 bits, at the sizes, masks and layouts where they can go wrong.

Rows are moved, not computed: copies, loads, stores, appended rows, bounds and the choice of
pages are compared for equality. Attention outputs, with u = finfo(type).eps / 2 the largest
relative error of one rounding, differ from the 64-bit ones by at most
  u |o|                    the output's own rounding, and
  (u + e) A + n 2^-25 |v|  with A = softmax . |V|: every probability is rounded to the type (u; in float16
                           those below 2^-14 by at most 2^-25 absolutely, and there are n of them), and
                           carries the relative error e of its exponent and of the sum it is divided by:
                           twice (d 2^-23 S + 2^-20), S = scale |q| . |k| the size of the terms of a score,
                           whose d products are added in 32 bits; 2^-20 covers the hardware's 2^x and
                           the sums of the parts' weights.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g).to(dtype)


def _ids(n, pool, seed):
    return torch.randperm(pool, generator=torch.Generator().manual_seed(seed))[:n].tolist()


def _bits(t):
    return t.contiguous().view(torch.int16)


def _key_bounds(k):
    """[..., rows, d] -> [..., 2, d]"""
    return torch.stack((k.amin(-2), k.amax(-2)), -2)


# ---------------------------------------------------------------- moving pages

@pytest.mark.parametrize("layers,hkv,page,d,dtype,n", [
    (1, 1, 16, 64, BF, 1), (28, 8, 64, 128, BF, 3), (3, 5, 32, 64, FP, 7), (2, 2, 256, 128, FP, 33), (1, 1, 16, 64, BF, 460)])
def test_copy_pages(layers, hkv, page, d, dtype, n):
    from megaqwen_amd import paged

    g = _gen(n)
    pool = 2 * n + 3
    k, v = _normal(g, (layers, pool, hkv, page, d), dtype), _normal(g, (layers, pool, hkv, page, d), dtype)
    b = _normal(g, (layers, pool, hkv, 2, d), dtype)
    ids = _ids(2 * n, pool, n)
    want = [t.clone() for t in (k, v, b)]
    for t in want:
        t[:, ids[n:]] = t[:, ids[:n]]
    paged.copy_pages(k, v, ids[:n], ids[n:], bounds=b)
    for got, w in zip((k, v, b), want):
        assert torch.equal(_bits(got), _bits(w))


def test_copy_pages_one_source_to_many_and_nothing():
    from megaqwen_amd import paged

    g = _gen(1)
    k, v = _normal(g, (2, 9, 3, 16, 64), BF), _normal(g, (2, 9, 3, 16, 64), BF)
    want = [t.clone() for t in (k, v)]
    for t in want:
        t[:, [1, 7, 3]] = t[:, 4:5]
    paged.copy_pages(k, v, [4, 4, 4], [1, 7, 3])
    assert all(torch.equal(_bits(a), _bits(w)) for a, w in zip((k, v), want))
    paged.copy_pages(k, v, [], [])
    assert all(torch.equal(_bits(a), _bits(w)) for a, w in zip((k, v), want))


@pytest.mark.parametrize("layers,hkv,page,d,dtype,n,extra", [
    (1, 1, 16, 64, BF, 1, 0), (2, 8, 64, 128, BF, 64, 5), (28, 8, 64, 128, BF, 333, 7), (3, 3, 128, 64, FP, 129, 1),
    (1, 2, 16, 128, FP, 16 * 450 + 3, 20), (2, 1, 256, 128, BF, 255, 0)])
def test_load_and_store_pages(layers, hkv, page, d, dtype, n, extra):
    from megaqwen_amd import paged

    g = _gen(n)
    used = -(-n // page)
    pool = used + 2
    k, v = _normal(g, (layers, pool, hkv, page, d), dtype), _normal(g, (layers, pool, hkv, page, d), dtype)
    b = torch.zeros(layers, pool, hkv, 2, d, dtype=dtype, device=DEV)
    kc, vc = _normal(g, (layers, hkv, n + extra, d), dtype), _normal(g, (layers, hkv, n + extra, d), dtype)
    ids = _ids(used, pool, n)
    want = [t.clone() for t in (k, v, b)]
    for i, p in enumerate(ids):
        m = min(page, n - i * page)
        for t, c in zip(want, (kc, vc)):
            t[:, p, :, :m] = c[:, :, i * page: i * page + m]
        want[2][:, p] = _key_bounds(kc[:, :, i * page: i * page + m])
    paged.load_pages(kc, vc, k, v, ids, n, bounds=b)
    for got, w in zip((k, v), want):
        assert torch.equal(_bits(got), _bits(w))  # (rows behind n, and the other pages, as they were)
    assert torch.equal(b, want[2])
    # and back into other caches: the same rows, the others as they were
    k2, v2 = _normal(g, tuple(kc.shape), dtype), _normal(g, tuple(kc.shape), dtype)
    want2 = [t.clone() for t in (k2, v2)]
    for t, c in zip(want2, (kc, vc)):
        t[:, :, :n] = c[:, :, :n]
    paged.store_pages(k, v, ids, n, k2, v2)
    for got, w in zip((k2, v2), want2):
        assert torch.equal(_bits(got), _bits(w))


def test_loaded_bounds_keep_infinities_and_nan_of_filled_rows_only():
    from megaqwen_amd import paged

    g = _gen(5)
    k, v = _normal(g, (1, 4, 1, 16, 64), BF), _normal(g, (1, 4, 1, 16, 64), BF)
    k[:, 2, :, 5:] = math.nan  # rows behind the loaded ones
    kc, vc = _normal(g, (1, 1, 30, 64), BF), _normal(g, (1, 1, 30, 64), BF)
    kc[0, 0, 3, 7], kc[0, 0, 4, 9], kc[0, 0, 2, 11] = math.inf, -math.inf, math.nan
    kc[0, 0, 21:] = math.nan
    b = torch.zeros(1, 4, 1, 2, 64, dtype=BF, device=DEV)
    paged.load_pages(kc, vc, k, v, [1, 2], 21, bounds=b)
    for page, rows in ((1, kc[0, 0, :16]), (2, kc[0, 0, 16:21])):
        want = _key_bounds(rows)
        assert torch.equal(b[0, page, 0].nan_to_num(nan=123.0, posinf=1e9, neginf=-1e9), want.nan_to_num(nan=123.0, posinf=1e9, neginf=-1e9))
    assert b[0, 1, 0].isnan().sum() == 2 and not b[0, 2].isnan().any()


@pytest.mark.parametrize("hkv,page,d,dtype,lens", [
    (8, 64, 128, BF, [0]), (8, 64, 128, BF, [0, 63, 64, 65, 200]), (3, 16, 64, FP, [15, 16, 17, 0, 31, 100, 1]),
    (16, 128, 128, FP, [127, 128, 5]), (40, 32, 64, BF, [33, 2])])
def test_append_rows(hkv, page, d, dtype, lens):
    from megaqwen_amd import paged

    g = _gen(len(lens) + hkv)
    B = len(lens)
    used = [n // page + 1 for n in lens]
    width, pool = max(used), sum(used) + 2
    order = _ids(pool, pool, 3)
    tables = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        tables[i, :n] = torch.tensor(order[at: at + n], dtype=torch.int32)
        at += n
    k, v = _normal(g, (pool, hkv, page, d), dtype), _normal(g, (pool, hkv, page, d), dtype)
    b = _key_bounds(k)
    # rows as a step's projections leave them, [kv heads, batch, d], and as a slice of wider rows
    kr = _normal(g, (hkv, B, d), dtype).transpose(0, 1)
    vr = _normal(g, (B, hkv, 2 * d), dtype)[:, :, d:]
    want = [t.clone() for t in (k, v, b)]
    for i, n in enumerate(lens):
        p, s = int(tables[i, n // page]), n % page
        want[0][p, :, s], want[1][p, :, s] = kr[i], vr[i]
        old = want[2][p]
        want[2][p] = torch.stack((kr[i], kr[i]), -2) if s == 0 else torch.stack(
            (torch.minimum(old[:, 0], kr[i]), torch.maximum(old[:, 1], kr[i])), -2)
    tables, lens_d = tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    paged.append_rows(kr, vr, k, v, tables, lens_d, bounds=b)
    for got, w in zip((k, v, b), want):
        assert torch.equal(_bits(got), _bits(w))
    assert lens_d.tolist() == lens


def test_append_rows_drops_rows_without_a_place():
    """A position behind the table, a negative one and pages outside the pool write nothing."""
    from megaqwen_amd import paged

    g = _gen(9)
    k, v = _normal(g, (4, 2, 16, 64), BF), _normal(g, (4, 2, 16, 64), BF)
    b = _key_bounds(k)
    before = [t.clone() for t in (k, v, b)]
    tables = torch.tensor([[0, 1], [0, 1], [-1, 0], [0, 4], [2, 2 ** 30]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([32, -1, 3, 17, 30], dtype=torch.int32, device=DEV)
    rows = _normal(g, (5, 2, 64), BF)
    paged.append_rows(rows, rows, k, v, tables, lens, bounds=b)
    assert all(torch.equal(_bits(a), _bits(w)) for a, w in zip((k, v, b), before))


# ---------------------------------------------------------------- attention

def _rows_of(pages, ids, h, n):
    """The first n rows of kv head h in pages `ids`, in 64 bits."""
    return pages[ids, h].reshape(-1, pages.shape[-1])[:n].double()


def _plain(q, k, v, scale):
    """(output, tolerance) of one query row [d] in 64 bits over rows [n, d]; zeros without rows."""
    u = torch.finfo(_plain.dtype).eps / 2
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    p = torch.softmax((k @ q) * scale, 0)
    o, a = p @ v, p @ v.abs()
    e = 2 * (q.numel() * 2.0 ** -23 * float((k.abs() @ q.abs()).max()) * scale + 2.0 ** -20)
    return o, u * o.abs() + (u + e) * a + k.shape[0] * 2.0 ** -25 * v.abs().amax(0)


def _check(out, q, rows_of, scale):
    """out [B, Hq, d] against the plain form; rows_of(b, kv head) gives (K, V)."""
    B, hq, d = q.shape
    _plain.dtype = q.dtype
    worst = 0.0
    for b in range(B):
        seen = {}
        for h in range(hq):
            j = h * rows_of.hkv // hq
            if j not in seen:
                seen[j] = rows_of(b, j)
            want, tol = _plain(q[b, h].double(), *seen[j], scale)
            diff = (out[b, h].double() - want).abs()
            assert bool((diff <= tol).all()), (b, h, float(diff.max()), float(tol[diff.argmax()]))
            worst = max(worst, float((diff / tol.clamp(min=1e-30)).max()))
    print(f"at most {worst:.2f} of the tolerance", flush=True)


def _setup(B, hkv, G, d, page, dtype, prefix, lens, seed=0, spare=2, kstd=1.0):
    g = _gen(seed)
    np_, used = -(-prefix // page), [-(-n // page) for n in lens]
    width, pool = max(1, *used), np_ + sum(used) + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tables = torch.full((B, width), -1, dtype=torch.int32)
    at = np_
    for b, n in enumerate(used):
        tables[b, :n] = order[at: at + n]
        at += n
    k, v = _normal(g, (pool, hkv, page, d), dtype, kstd), _normal(g, (pool, hkv, page, d), dtype, 0.64)
    q = _normal(g, (B, hkv * G, d), dtype)
    pre = order[:np_]
    # nothing behind the last row may reach an output
    for ids, n in [(pre, prefix)] + [(tables[b, :u], n) for b, (u, n) in enumerate(zip(used, lens))]:
        if n % page:
            k[int(ids[-1]), :, n % page:] = math.nan
            v[int(ids[-1]), :, n % page:] = math.inf
    for p in order[at:].tolist():
        k[p], v[p] = math.nan, math.nan

    def rows_of(b, j):
        own = tables[b, :used[b]].long()
        return tuple(torch.cat((_rows_of(t, pre.long(), j, prefix), _rows_of(t, own, j, lens[b]))) for t in (k, v))

    rows_of.hkv = hkv
    return q, k, v, pre.to(DEV), tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), rows_of


SHARED = [
    # batch, kv heads, queries a kv head, d, page, type, prefix, own rows
    (1, 8, 2, 128, 64, BF, 0, [1]),
    (1, 8, 2, 128, 64, BF, 1, [0]),
    (1, 1, 1, 64, 16, FP, 0, [33]),
    (3, 8, 2, 128, 64, BF, 0, [0, 5, 0]),
    (2, 8, 2, 128, 64, BF, 64, [64, 128]),
    (4, 8, 2, 128, 64, BF, 512, [37, 1, 64, 20]),
    (9, 8, 2, 128, 64, BF, 1000, [300, 0, 17, 129, 64, 63, 65, 1, 200]),
    (17, 2, 1, 128, 16, FP, 777, list(range(0, 17 * 9, 9))),
    (23, 4, 5, 64, 16, FP, 1117, [(37 * i) % 301 for i in range(23)]),
    (5, 3, 7, 64, 32, BF, 95, [31, 32, 33, 0, 700]),
    (2, 1, 16, 128, 128, BF, 2049, [1025, 127]),
    (2, 2, 20, 128, 256, FP, 255, [257, 511]),
    (33, 1, 4, 128, 16, BF, 31, [i % 3 for i in range(33)]),
    (70, 8, 2, 128, 64, BF, 300, [(11 * i) % 90 for i in range(70)]),
    (1, 8, 2, 128, 16, BF, 0, [9000]),
    (1, 8, 2, 64, 16, FP, 9001, [40]),
    (65, 1, 8, 64, 64, BF, 4000, [i for i in range(65)]),
    (40, 8, 2, 128, 64, BF, 4000, [(13 * i) % 65 for i in range(40)]),
    (32, 8, 1, 128, 32, FP, 500, [(29 * i) % 130 for i in range(32)]),
    (33, 8, 1, 128, 32, FP, 500, [(29 * i) % 130 for i in range(33)]),
    (6, 2, 2, 64, 16, BF, 601, [39, 0, 20, 1, 38, 16]),
    (6, 2, 2, 64, 16, BF, 609, [39, 0, 20, 1, 38, 16]),
    (130, 2, 1, 128, 64, BF, 200, [0] * 130),
    (70, 2, 2, 128, 32, FP, 900, [(17 * i) % 200 for i in range(70)]),
    (40, 1, 4, 128, 256, BF, 1500, [(91 * i) % 600 for i in range(40)]),
]


@pytest.mark.parametrize("case", SHARED, ids=lambda c: f"b{c[0]}h{c[1]}x{c[2]}d{c[3]}p{c[4]}-{c[6]}")
def test_shared_prefix_attention(case):
    from megaqwen_amd import paged

    B, hkv, G, d, page, dtype, prefix, lens = case
    q, k, v, pre, tables, lens_d, rows_of = _setup(*case, seed=B + prefix)
    scale = 1 / math.sqrt(d)
    out = paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d)
    assert out.shape == q.shape and out.dtype == dtype
    _check(out, q, rows_of, scale)
    for b, n in enumerate(lens):
        if n + prefix == 0:
            assert torch.equal(out[b], torch.zeros_like(out[b]))
    # a length to lay the work out for, right or wrong, changes the order of the sums only
    for hint in (1, max(1, max(lens))):
        _check(paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d, max_len=hint), q, rows_of, scale)


@pytest.mark.parametrize("case", [
    # tiles of 128 rows: more than 1024 steps of 64 keys by 128 rows, with a last tile, page, part and step that are not full
    (40, 16, 4, 128, 64, BF, 2100, [0, 1, 63, 64, 65, 300, 7, 129] * 5),
    (30, 16, 5, 64, 16, FP, 2113, [0, 200, 16] * 10),
    (65, 8, 2, 128, 256, FP, 4097, [0] * 65),
    (65, 16, 2, 64, 128, BF, 2100, [40] * 65),
], ids=lambda c: f"b{c[0]}h{c[1]}x{c[2]}d{c[3]}p{c[4]}n{c[6]}")
def test_shared_prefix_attention_of_large_batches(case):
    from megaqwen_amd import paged

    B, hkv, G, d, page, dtype, prefix, lens = case
    q, k, v, pre, tables, lens_d, rows_of = _setup(B, hkv, G, d, page, dtype, prefix, lens, seed=B)
    out = paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d)
    _check(out, q, rows_of, 1 / math.sqrt(d))


@pytest.mark.parametrize("case", [
    # more than 512 sequences times kv heads with at most 256 own rows: a wave a sequence
    (130, 4, 2, 128, 64, BF, 0, [0, 1, 31, 32, 33, 64, 100, 256, 255, 129]),
    (130, 4, 2, 128, 64, BF, 70, [0, 1, 31, 32, 33, 64, 100, 256, 255, 129]),
    (65, 8, 17, 64, 16, FP, 300, [0, 16, 17, 200]),
    (515, 1, 1, 128, 32, FP, 1500, [5]),
    (103, 5, 3, 64, 256, BF, 0, [0, 0, 7]),
], ids=lambda c: f"b{c[0]}h{c[1]}x{c[2]}d{c[3]}p{c[4]}n{c[6]}")
def test_shared_prefix_attention_of_many_short_sequences(case):
    from megaqwen_amd import paged

    B, hkv, G, d, page, dtype, prefix, some = case
    lens = (some * B)[:B]
    q, k, v, pre, tables, lens_d, rows_of = _setup(B, hkv, G, d, page, dtype, prefix, lens, seed=B)
    out = paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d, max_len=max(lens))
    _check(out, q, rows_of, 1 / math.sqrt(d))
    # laid out for fewer rows than there are, and (a workgroup a sequence) for more
    for max_len in (1, 300):
        _check(paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d, max_len=max_len), q, rows_of, 1 / math.sqrt(d))
    # a page outside the pool is its own sequence's matter only
    at = next(b for b in range(9, B) if lens[b] > 0)
    tables[at, 0] = k.shape[0]
    bad = paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d, max_len=max(lens))
    assert bool(bad[at].isnan().all())
    others = [b for b in range(B) if b != at]
    assert torch.equal(_bits(bad[others]), _bits(out[others]))


def test_sparse_attention_of_many_short_choices():
    """More than 512 sequences times kv heads, of which each reads at most 256 rows."""
    from megaqwen_amd import paged

    B, hkv, G, d, page, top = 140, 4, 2, 64, 32, 8
    lens = ([0, 1, 256, 255, 900, 1000, 33] * B)[:B]
    q, k, v, _, tables, lens_d, _ = _setup(B, hkv, G, d, page, BF, 0, lens, seed=8)
    bounds = torch.zeros(k.shape[0], hkv, 2, d, dtype=BF, device=DEV)
    host = tables.cpu().long()
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            bounds[host[b, i]] = _key_bounds(k[host[b, i], :, : min(page, n - i * page)])
    out, chosen = paged.sparse_attention(q, k, v, bounds, tables, lens_d, top)
    want = {(b, j): _plain_choice(q[b, j * G:(j + 1) * G], bounds[:, j], host[b], lens[b], page, top) for b in range(B) for j in range(hkv)}
    for (b, j), sel in want.items():
        assert chosen[b, j].tolist() == sel + [-1] * (top - len(sel))

    def rows_of(b, j):
        sel = want[b, j]
        n = 0 if not sel else (len(sel) - 1) * page + (lens[b] - 1) % page + 1
        return tuple(_rows_of(t, host[b][sel], j, n) for t in (k, v))

    rows_of.hkv = hkv
    _check(out, q, rows_of, 1 / math.sqrt(d))


def test_shared_prefix_attention_strides_scale_and_out():
    """q and out as slices of wider rows, tables as a slice of whole tables, another scale; repeats are bit-identical."""
    from megaqwen_amd import paged

    B, hkv, G, d, page = 6, 4, 3, 128, 32
    lens = [40, 0, 96, 7, 64, 33]
    q, k, v, pre, tables, lens_d, rows_of = _setup(B, hkv, G, d, page, BF, 130, lens, seed=4)
    wide = torch.zeros(B, hkv * G + 5, d + 64, dtype=BF, device=DEV)
    wide[:, 2:2 + hkv * G, 32:32 + d] = q
    whole = torch.cat((pre.view(1, -1).expand(B, -1), tables), 1).contiguous()
    out = torch.full((hkv * G, B, d), 7.0, dtype=BF, device=DEV)
    got = paged.shared_prefix_attention(wide[:, 2:2 + hkv * G, 32:32 + d], k, v, whole[0, :pre.numel()], 130, whole[:, pre.numel():],
                                        lens_d, scale=0.3, out=out.transpose(0, 1))
    assert got.data_ptr() == out.data_ptr()
    _check(got, q, rows_of, 0.3)
    again = paged.shared_prefix_attention(q, k, v, pre, 130, tables, lens_d, scale=0.3)
    assert torch.equal(_bits(again), _bits(got))


def test_query_layouts_that_torch_allows():
    """Heads before the batch, the same query for all (stride 0), one sequence or one head with a stride that is never used."""
    from megaqwen_amd import paged

    for B, hkv, G, make in (
            (5, 2, 3, lambda q: q.transpose(0, 1).contiguous().transpose(0, 1)), (4, 2, 2, lambda q: q[:1].expand(4, -1, -1)),
            (1, 2, 2, lambda q: q.as_strided(q.shape, (3, q.stride(1), 1))), (3, 1, 1, lambda q: q.as_strided(q.shape, (q.stride(0), 5, 1)))):
        for prefix in (40, 900):  # (one launch, and two)
            q, k, v, pre, tables, lens_d, rows_of = _setup(B, hkv, G, 64, 16, BF, prefix, [30 + b for b in range(B)], seed=B)
            q = make(q)
            _check(paged.shared_prefix_attention(q, k, v, pre, prefix, tables, lens_d), q, rows_of, 1 / 8)


def test_attention_of_large_scores_and_one_sided_values():
    """Scores of hundreds (one key takes all) and values of one sign: no overflow, no bias."""
    from megaqwen_amd import paged

    q, k, v, pre, tables, lens_d, rows_of = _setup(3, 2, 2, 128, 64, BF, 700, [90, 0, 200], seed=8, kstd=30.0)
    v.copy_(torch.where(v.isfinite(), v.abs(), v))
    out = paged.shared_prefix_attention(q, k, v, pre, 700, tables, lens_d)
    _check(out, q, rows_of, 1 / math.sqrt(128))


def test_attention_names_a_page_outside_the_pool():
    """A sequence that needs one gets NaN, the others are as without it; a bad prefix page reaches all."""
    from megaqwen_amd import paged

    q, k, v, pre, tables, lens_d, rows_of = _setup(4, 2, 2, 64, 16, BF, 50, [20, 40, 60, 33], seed=2)
    good = paged.shared_prefix_attention(q, k, v, pre, 50, tables, lens_d)
    for bad_id in (-1, k.shape[0], 2 ** 31 - 1):
        t = tables.clone()
        t[2, 1] = bad_id
        out = paged.shared_prefix_attention(q, k, v, pre, 50, t, lens_d)
        assert bool(out[2].isnan().all())
        keep = [0, 1, 3]
        assert torch.equal(_bits(out[keep]), _bits(good[keep]))
    p = pre.clone()
    p[3] = k.shape[0]
    assert bool(paged.shared_prefix_attention(q, k, v, p, 50, tables, lens_d).isnan().all())
    # lengths outside the table count as none and as all of it
    over = torch.tensor([-5, 1000, 60, 33], dtype=torch.int32, device=DEV)
    t = tables.clone()
    t[1] = tables[2]
    k2, v2 = torch.where(k.isnan(), 0, k), torch.where(v.isfinite(), v, 0)
    out = paged.shared_prefix_attention(q, k2, v2, pre, 50, t, over)
    full = paged.shared_prefix_attention(q, k2, v2, pre, 50, t, torch.tensor([0, 64, 60, 33], dtype=torch.int32, device=DEV))
    assert torch.equal(_bits(out), _bits(full))


def test_long_pool_passes_32_bit_offsets():
    """Pages whose byte offsets in the pool need more than 32 bits."""
    from megaqwen_amd import paged

    pages, hkv, page, d = 40000, 8, 64, 128  # 2.6e9 elements, 5.2 GB each for K and V
    k = torch.zeros(pages, hkv, page, d, dtype=BF, device=DEV)
    v = torch.zeros(pages, hkv, page, d, dtype=BF, device=DEV)
    g = _gen(3)
    ids = [39999, 33000, 1, 39998]
    for i in ids:
        k[i], v[i] = _normal(g, (hkv, page, d), BF), _normal(g, (hkv, page, d), BF)
    q = _normal(g, (1, 16, d), BF)
    tables, lens = torch.tensor([ids[1:]], dtype=torch.int32, device=DEV), torch.tensor([150], dtype=torch.int32, device=DEV)

    def rows_of(b, j):
        return tuple(torch.cat((_rows_of(t, ids[:1], j, 60), _rows_of(t, ids[1:], j, 150))) for t in (k, v))

    rows_of.hkv = hkv
    _check(paged.shared_prefix_attention(q, k, v, torch.tensor(ids[:1], dtype=torch.int32, device=DEV), 60, tables, lens), q, rows_of,
           1 / math.sqrt(d))
    row = _normal(g, (1, hkv, d), BF)
    paged.append_rows(row, row, k, v, tables, lens)
    assert torch.equal(k[39998, :, 150 - 128], row[0]) and torch.equal(v[39998, :, 150 - 128], row[0])
    paged.copy_pages(k[None], v[None], [39998, 33000], [39997, 2])
    assert torch.equal(k[39997], k[39998]) and torch.equal(v[2], v[33000])


# ---------------------------------------------------------------- choosing pages

def _plain_choice(q, bounds, ids, n, page, top):
    """Pages chosen for the queries [G, d] of one kv head, from bounds [pages, 2, d]."""
    used = -(-n // page)
    if used <= top:
        return list(range(used))
    lo, hi = bounds[ids[:used]].double().unbind(1)
    s = torch.maximum(q.double()[None] * lo[:, None], q.double()[None] * hi[:, None]).sum((1, 2)).tolist()
    best = sorted(range(used - 1), key=lambda i: (-s[i], i))[: top - 1]
    return sorted(best + [used - 1])


SPARSE = [
    # batch, kv heads, queries a kv head, d, page, type, rows, top
    (1, 8, 2, 128, 64, BF, [1], 1),
    (1, 8, 2, 128, 64, BF, [2000], 8),
    (4, 8, 2, 128, 64, BF, [0, 64, 65, 700], 2),
    (3, 2, 5, 64, 16, FP, [400, 33, 1000], 1),
    (3, 2, 5, 64, 16, FP, [400, 33, 1000], 7),
    (2, 4, 16, 128, 32, BF, [1500, 999], 24),
    (2, 1, 3, 64, 128, FP, [5000, 4999], 40),
    (1, 1, 1, 64, 16, BF, [16 * 3000 + 5], 1500),
    (5, 3, 20, 64, 16, BF, [161, 160, 159, 17, 16], 5),
]


@pytest.mark.parametrize("case", SPARSE, ids=lambda c: f"b{c[0]}h{c[1]}x{c[2]}d{c[3]}p{c[4]}n{c[6][0]}t{c[7]}")
def test_sparse_attention(case):
    from megaqwen_amd import paged

    B, hkv, G, d, page, dtype, lens, top = case
    q, k, v, _, tables, lens_d, _ = _setup(B, hkv, G, d, page, dtype, 0, lens, seed=B + top)
    bounds = torch.zeros(k.shape[0], hkv, 2, d, dtype=dtype, device=DEV)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            p = int(tables[b, i])
            bounds[p] = _key_bounds(k[p, :, : min(page, n - i * page)])
    out, chosen = paged.sparse_attention(q, k, v, bounds, tables, lens_d, top)
    assert chosen.shape == (B, hkv, top) and chosen.dtype == torch.int32
    host = tables.cpu().long()
    want = {}
    for b in range(B):
        for j in range(hkv):
            want[b, j] = _plain_choice(q[b, j * G:(j + 1) * G], bounds[:, j], host[b], lens[b], page, top)
            assert chosen[b, j].tolist() == want[b, j] + [-1] * (top - len(want[b, j]))

    def rows_of(b, j):
        sel = want[b, j]
        n = 0 if not sel else (len(sel) - 1) * page + (lens[b] - 1) % page + 1
        return tuple(_rows_of(t, host[b][sel], j, n) for t in (k, v))

    rows_of.hkv = hkv
    _check(out, q, rows_of, 1 / math.sqrt(d))


@pytest.mark.parametrize("G,d", [(20, 128), (1, 64), (33, 64)])
def test_sparse_parts_join_in_a_replayed_graph(G, d):
    """Sequences of no, one and many parts, whose lengths change between the replays of one graph; all pages are chosen."""
    from megaqwen_amd import paged

    hkv, page, top = 2, 64, 47
    lens = [3000, 128, 129, 1500, 3000, 1]
    q, k, v, _, tables, lens_d, rows_of = _setup(6, hkv, G, d, page, BF, 0, lens, seed=G)
    bounds = torch.zeros(k.shape[0], hkv, 2, d, dtype=BF, device=DEV)  # (never decides: no sequence has more pages)

    def eager():
        return paged.sparse_attention(q, k, v, bounds, tables, lens_d, top)[0]

    _check(eager(), q, rows_of, 1 / math.sqrt(d))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [eager() for _ in range(3)]
    for now in (lens, [0, 100, 128, 700, 2999, 1], [1280, 1, 0, 1408, 64, 0], lens):
        lens_d.copy_(torch.tensor(now, dtype=torch.int32))
        want = eager().clone()
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(_bits(o), _bits(want))
        for b, n in enumerate(now):
            assert n > 0 or not want[b].any()
    _check(want, q, rows_of, 1 / math.sqrt(d))


def test_sparse_choice_of_equal_scores_takes_the_earlier_pages():
    from megaqwen_amd import paged

    g = _gen(6)
    B, hkv, G, d, page, pages, top = 2, 2, 2, 64, 16, 1200, 500
    k, v = _normal(g, (pages, hkv, page, d), BF), _normal(g, (pages, hkv, page, d), BF)
    q = _normal(g, (B, hkv * G, d), BF)
    two = _key_bounds(_normal(g, (2, hkv, page, d), BF))
    bounds = two[torch.arange(pages, device=DEV) % 3 % 2].contiguous()  # three pages, two kinds
    tables = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(B, 1)
    lens = torch.tensor([page * pages, page * 900 + 1], dtype=torch.int32, device=DEV)
    _, chosen = paged.sparse_attention(q, k, v, bounds, tables, lens, top)
    for b, n in enumerate(lens.tolist()):
        for j in range(hkv):
            assert chosen[b, j].tolist() == _plain_choice(q[b, j * G:(j + 1) * G], bounds[:, j], list(range(pages)), n, page, top)
    # all equal, and all zero (of either sign)
    for value in (1.0, 0.0, -0.0):
        _, chosen = paged.sparse_attention(q, k, v, torch.full_like(bounds, value), tables, lens, top)
        for b, n in enumerate(lens.tolist()):
            want = list(range(top - 1)) + [-(-n // page) - 1]
            assert all(chosen[b, j].tolist() == want for j in range(hkv))


def test_sparse_widest_table():
    from megaqwen_amd import _abi, paged

    g = _gen(7)
    width, top = _abi.MQ_MAX_TABLE_WIDTH, 9
    k, v = _normal(g, (50, 1, 16, 64), BF), _normal(g, (50, 1, 16, 64), BF)
    bounds, q = _key_bounds(k), _normal(g, (1, 2, 64), BF)
    tables = torch.randint(0, 50, (1, width), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    lens = torch.tensor([16 * width], dtype=torch.int32, device=DEV)
    out, chosen = paged.sparse_attention(q, k, v, bounds, tables.to(DEV), lens, top)
    want = _plain_choice(q[0], bounds[:, 0], tables[0].long(), 16 * width, 16, top)
    assert chosen[0, 0].tolist() == want

    def rows_of(b, j):
        return tuple(_rows_of(t, tables[0].long()[want], 0, 16 * top) for t in (k, v))

    rows_of.hkv = 1
    _check(out, q, rows_of, 1 / 8)


def test_sparse_page_outside_the_pool():
    from megaqwen_amd import paged

    q, k, v, _, tables, lens_d, _ = _setup(2, 2, 2, 64, 16, BF, 0, [300, 301], seed=3)
    bounds = _key_bounds(torch.where(k.isnan(), 0, k))
    good, chosen = paged.sparse_attention(q, k, v, bounds, tables, lens_d, 4)
    tables[1, 7] = k.shape[0] + 5
    out, _ = paged.sparse_attention(q, k, v, bounds, tables, lens_d, 4)
    assert torch.equal(_bits(out[0]), _bits(good[0])) and bool(out[1].isnan().all())


# ---------------------------------------------------------------- streams, graphs, devices

def test_operators_in_a_captured_graph():
    """append, shared and sparse attention captured once and replayed over changing contents, with eager
    calls between the replays: every replay equals the eager result."""
    from megaqwen_amd import paged

    B, hkv, G, d, page = 3, 8, 2, 128, 64
    q, k, v, pre, tables, lens, _ = _setup(B, hkv, G, d, page, BF, 200, [100, 64, 300], seed=1)
    k, v = torch.where(k.isnan(), 0, k), torch.where(v.isfinite(), v, 0)
    tables = tables.clamp(min=0)
    bounds = _key_bounds(k)
    row = _normal(_gen(5), (B, hkv, d), BF)

    def step():
        paged.append_rows(row, row, k, v, tables, lens, bounds=bounds)
        return (paged.shared_prefix_attention(q, k, v, pre, 200, tables, lens),) + paged.sparse_attention(q, k, v, bounds, tables, lens, 2)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same calls
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    g = _gen(17)
    for i in range(4):
        q.copy_(_normal(g, tuple(q.shape), BF))
        row.copy_(_normal(g, tuple(row.shape), BF))
        lens.copy_(torch.tensor([100 + i, 64 + 30 * i, 300 - 50 * i], dtype=torch.int32))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for graph, outs in graphs:
            for t in outs:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert torch.equal(_bits(outs[0]), _bits(want[0])) and torch.equal(_bits(outs[1]), _bits(want[1]))
            assert torch.equal(outs[2], want[2])


def test_operators_on_two_streams_at_once():
    from megaqwen_amd import paged

    a = _setup(8, 8, 2, 128, 64, BF, 2000, [200] * 8, seed=1)
    b = _setup(5, 4, 3, 64, 16, FP, 900, [70] * 5, seed=2)

    def call(s, n):
        return paged.shared_prefix_attention(s[0], s[1], s[2], s[3], n, s[4], s[5])

    want = call(a, 2000), call(b, 900)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        for stream, s, n in zip(streams, (a, b), (2000, 900)):
            with torch.cuda.stream(stream):
                got.append(call(s, n))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(_bits(o), _bits(want[i % 2]))
