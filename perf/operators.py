"""The operators on a paged K/V cache, as cases that can be timed and compared.

A pool holds K and V rows in pages, [layers, pages, kv heads, page size, head dim], and every
sequence has a table of page ids, so that sequences that begin alike share pages. The operators:

- "copy": whole pages of every layer to other pages (a fork's private last page; compaction);
- "load" / "store": positions of a contiguous cache [layers, kv heads, positions, head dim], as the
  prefill and the decode step use it, into pages and back; loading also gives each page's bounds,
  the least and the greatest key entry of every head and dim over the page's filled rows;
- "append": one new K and V row a sequence behind the rows that it has, and the bounds;
- "shared": one query token a sequence over a prefix that all sequences share and over the
  sequence's own rows behind it;
- "sparse": one query token a sequence over its last page and the pages whose bounds allow the
  largest scores.

K rows are RMS-normalised and rotated, so their entries are N(0, 1), and so are a query's; V rows are
a projection of normalised rows, N(0, 0.64). Pages that no sequence uses hold rows of earlier ones.
"""

import math

import torch

own = False

V_STD = 0.64  # 0.02 * sqrt(1024)
# the package's model: 28 layers, 8 kv heads with 2 query heads each, heads of 128
MODEL = {"layers": 28, "hkv": 8, "g": 2, "d": 128, "dtype": "bf16"}
LAYER = {"layers": 1, "hkv": 8, "g": 2, "d": 128, "dtype": "bf16"}


def listed():
    return [
        # a second answer to a prompt: its unfilled last page becomes private
        {"name": "copy_fork1", "op": "copy", **MODEL, "page": 16, "pool": 40, "n": 1},
        # a pool that has emptied in places is closed up
        {"name": "copy_compact120", "op": "copy", **MODEL, "page": 64, "pool": 300, "n": 120},
        # a prefilled prompt of a few pages of text, of no round length, goes into the pool
        {"name": "load_s3000", "op": "load", **MODEL, "page": 64, "pool": 64, "n": 3000},
        # one of the answers goes on alone, in the cache of the batch-1 decoder
        {"name": "store_s1117", "op": "store", **MODEL, "page": 64, "pool": 64, "n": 1117},
        # a decode step of one sequence: one row of one layer, the smallest call
        {"name": "append_b1", "op": "append", **LAYER, "page": 64, "pool": 8, "batch": 1, "own": 200},
        # a decode step of a large batch
        {"name": "append_b200", "op": "append", **LAYER, "page": 64, "pool": 1500, "batch": 200, "own": 511},
        # four answers to a question of a few lines, in their first words
        {"name": "shared_b4_p512", "op": "shared", **LAYER, "page": 64, "batch": 4, "prefix": 512, "own": 37, "empty": False},
        # sixty-four answers behind a long document
        {"name": "shared_b64_p8192", "op": "shared", **LAYER, "page": 64, "batch": 64, "prefix": 8192, "own": 512, "empty": False},
        # heads of 64, five to a kv head, in half precision; an odd batch, some sequences with no rows of their own
        {"name": "shared_b23_p1117_fp16", "op": "shared", "layers": 1, "hkv": 4, "g": 5, "d": 64, "dtype": "fp16", "page": 16,
         "batch": 23, "prefix": 1117, "own": 300, "empty": True},
        # the largest batch behind the longest context, long answers
        {"name": "shared_b256_p15001", "op": "shared", **LAYER, "page": 64, "batch": 256, "prefix": 15001, "own": 1024, "empty": False},
        # one long context, an eighth of its pages read
        {"name": "sparse_b1_s16000", "op": "sparse", **LAYER, "page": 64, "batch": 1, "own": 16000, "top": 32},
        # many long contexts at once
        {"name": "sparse_b32_s16000", "op": "sparse", **LAYER, "page": 64, "batch": 32, "own": 16000, "top": 32},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["copy", "load", "store", "append", "shared", "shared", "shared", "sparse", "sparse"])
    heads = {"hkv": rng.choice([1, 2, 4, 8, 8]), "g": rng.choice([1, 2, 2, 3, 4, 5, 7, 8, 16]), "d": rng.choice([64, 128, 128]),
             "dtype": rng.choice(["bf16", "bf16", "fp16"]), "page": rng.choice([16, 32, 64, 64, 128])}
    if op == "copy":
        n = _spread(rng, 1, 120)
        return {"op": op, "layers": rng.randint(1, 28), **heads, "page": rng.choice([16, 32, 64]), "pool": 2 * n + rng.randint(0, 50), "n": n}
    if op in ("load", "store"):
        n = _spread(rng, 1, 3000)
        return {"op": op, "layers": rng.randint(1, 28), **heads, "pool": -(-n // heads["page"]) + rng.randint(0, 20), "n": n}
    if op == "append":
        batch, own_rows = _spread(rng, 1, 200), _spread(rng, 1, 500)
        return {"op": op, "layers": 1, **heads, "pool": batch * (own_rows // heads["page"] + 1) + rng.randint(0, 20), "batch": batch, "own": own_rows}
    if op == "shared":
        return {"op": op, "layers": 1, **heads, "batch": _spread(rng, 1, 256 * 2 // max(2, heads["g"])),
                "prefix": rng.choice([0, _spread(rng, 1, 15000), _spread(rng, 1, 15000)]), "own": _spread(rng, 1, 1024), "empty": rng.random() < 0.5}
    return {"op": op, "layers": 1, **heads, "batch": _spread(rng, 1, 32 * 2 // max(2, heads["g"])), "own": _spread(rng, 1, 16000),
            "top": _spread(rng, 1, max(1, 2048 // heads["page"]))}


def _lens(case):
    """Rows that each sequence of a batch has of its own: spread over 1 .. own (the first has them
    all), every third one none where the case says so."""
    n = [max(1, round(case["own"] * (1 - (b * 0.6180339887) % 1))) for b in range(case["batch"])]
    return [0 if case.get("empty") and b % 3 == 1 else x for b, x in enumerate(n)]


def _pages(rows, page):
    return -(-rows // page)


def _type(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]


def _normal(case, g, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).to(_type(case))


def _bounds(k_pages):
    """[..., page, d] -> [..., 2, d]: the bounds of whole pages."""
    return torch.stack((k_pages.amin(-2), k_pages.amax(-2)), -2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)  # for what the host decides
    L, hkv, d, page = case["layers"], case["hkv"], case["d"], case["page"]
    s = {"case": case}
    if case["op"] in ("copy", "load", "store"):
        pool = (L, case["pool"], hkv, page, d)
        s["k_pages"], s["v_pages"] = _normal(case, g, pool), _normal(case, g, pool, V_STD)
        order = torch.randperm(case["pool"], generator=h).tolist()
        if case["op"] == "copy":
            s["src"], s["dst"] = order[: case["n"]], order[case["n"]: 2 * case["n"]]
            s["bounds"] = _bounds(s["k_pages"])
        else:
            s["pages"] = order[: _pages(case["n"], page)]
            cache = (L, hkv, case["n"] + 100, d)
            s["k_cache"], s["v_cache"] = _normal(case, g, cache), _normal(case, g, cache, V_STD)
            s["bounds"] = torch.zeros(L, case["pool"], hkv, 2, d, dtype=_type(case), device="cuda")
        return s
    lens, prefix = _lens(case), case.get("prefix", 0)
    rows = [n + 1 for n in lens] if case["op"] == "append" else lens
    used = [_pages(n, page) for n in rows]
    width, shared = max(1, max(used)), _pages(prefix, page)
    pool = max(case.get("pool", 0), shared + sum(used) + 3)
    s["k_pages"], s["v_pages"] = _normal(case, g, (pool, hkv, page, d)), _normal(case, g, (pool, hkv, page, d), V_STD)
    order = torch.randperm(pool, generator=h).to(torch.int32)
    tables = torch.full((case["batch"], width), -1, dtype=torch.int32)
    at = shared
    for b, n in enumerate(used):
        tables[b, :n] = order[at: at + n]
        at += n
    s["tables"], s["lens"] = tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    s["scale"] = 1.0 / math.sqrt(d)
    if case["op"] == "append":
        s["k"], s["v"] = _normal(case, g, (case["batch"], hkv, d)), _normal(case, g, (case["batch"], hkv, d), V_STD)
        s["bounds"] = _bounds(s["k_pages"])
        return s
    s["q"] = _normal(case, g, (case["batch"], hkv * case["g"], d))
    if case["op"] == "shared":
        s["prefix_pages"], s["prefix_len"] = order[:shared].cuda(), prefix
    else:
        # the bounds of a page take in its filled rows only
        s["bounds"] = _bounds(s["k_pages"])
        b = torch.arange(case["batch"], device="cuda")
        last = s["tables"][b, ((s["lens"] - 1) // page).long()].long()
        filled = ((s["lens"] - 1) % page + 1).view(-1, 1, 1, 1)
        out = torch.arange(page, device="cuda").view(1, 1, -1, 1) >= filled
        rows = s["k_pages"][last]
        s["bounds"][last] = torch.stack((rows.masked_fill(out, math.inf).amin(-2), rows.masked_fill(out, -math.inf).amax(-2)), -2)
    return s


# ---- the plain forms

def _plain_load(s):
    n, page = s["case"]["n"], s["case"]["page"]
    pages = torch.tensor(s["pages"], device="cuda")
    at = torch.arange(n, device="cuda")
    where = (slice(None), pages[at // page], slice(None), at % page)
    s["k_pages"][where] = s["k_cache"][:, :, :n].permute(2, 0, 1, 3)
    s["v_pages"][where] = s["v_cache"][:, :, :n].permute(2, 0, 1, 3)
    rows = s["k_pages"][:, pages]
    filled = (torch.arange(pages.numel(), device="cuda") * page).view(-1, 1, 1, 1) + torch.arange(page, device="cuda").view(1, 1, -1, 1) < n
    s["bounds"][:, pages] = torch.stack((rows.masked_fill(~filled, math.inf).amin(-2), rows.masked_fill(~filled, -math.inf).amax(-2)), -2)
    return s["k_pages"], s["v_pages"], s["bounds"]


def _plain_store(s):
    n, page = s["case"]["n"], s["case"]["page"]
    pages = torch.tensor(s["pages"], device="cuda")
    at = torch.arange(n, device="cuda")
    where = (slice(None), pages[at // page], slice(None), at % page)
    s["k_cache"][:, :, :n] = s["k_pages"][where].permute(1, 2, 0, 3)
    s["v_cache"][:, :, :n] = s["v_pages"][where].permute(1, 2, 0, 3)
    return s["k_cache"], s["v_cache"]


def _plain_append(s):
    page, lens = s["case"]["page"], s["lens"].long()
    b = torch.arange(lens.numel(), device="cuda")
    pages, slot = s["tables"][b, lens // page].long(), lens % page
    s["k_pages"][pages, :, slot] = s["k"]
    s["v_pages"][pages, :, slot] = s["v"]
    before, first = s["bounds"][pages], (slot == 0).view(-1, 1, 1)
    lo, hi = torch.minimum(before[:, :, 0], s["k"]), torch.maximum(before[:, :, 1], s["k"])
    s["bounds"][pages] = torch.stack((torch.where(first, s["k"], lo), torch.where(first, s["k"], hi)), -2)
    return s["k_pages"], s["v_pages"], s["bounds"]


def _softmax(x):
    """exp(x - max) over the last axis and its sum; a row without a finite value gives zeros."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    return p, p.sum(-1, keepdim=True)


def _plain_shared(s):
    c = s["case"]
    B, hkv, G, d, n = c["batch"], c["hkv"], c["g"], c["d"], s["prefix_len"]
    q = s["q"].float().view(B, hkv, G, d)
    rows = lambda pages: pages.float().transpose(-4, -3).flatten(-3, -2)  # [.., pages, h, page, d] -> [.., h, rows, d]  # noqa: E731
    kp, vp = (rows(t[s["prefix_pages"].long()])[:, :n].contiguous() for t in (s["k_pages"], s["v_pages"]))
    tables = s["tables"].clamp(min=0).long()
    ko, vo = rows(s["k_pages"][tables]), rows(s["v_pages"][tables])
    has = torch.arange(ko.shape[2], device="cuda").view(1, 1, 1, -1) < s["lens"].view(-1, 1, 1, 1)
    sp = (q.transpose(0, 1).reshape(hkv, B * G, d) @ kp.transpose(1, 2).contiguous()).view(hkv, B, G, n).transpose(0, 1)
    so = (q @ ko.transpose(2, 3).contiguous()).masked_fill(~has, -math.inf)
    p, total = _softmax(torch.cat((sp, so), -1) * s["scale"])
    o = (p[..., :n].transpose(0, 1).reshape(hkv, B * G, n) @ vp).view(hkv, B, G, d).transpose(0, 1)
    o = o + p[..., n:] @ vo.masked_fill(~has.transpose(2, 3), 0.0)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.reshape(B, hkv * G, d).to(s["q"].dtype)


def _plain_sparse(s):
    c = s["case"]
    B, hkv, G, d, page, top = c["batch"], c["hkv"], c["g"], c["d"], c["page"], c["top"]
    tables, lens = s["tables"].clamp(min=0).long(), s["lens"].long()
    # scores in 64 bits: a page on the border of the choice has to fall on the same side everywhere
    q = s["q"].double().view(B, 1, hkv, G, d)
    lo, hi = s["bounds"][tables].double().unsqueeze(3).unbind(4)
    score = torch.maximum(q * lo, q * hi).sum((3, 4)).transpose(1, 2)  # [B, hkv, pages]
    at, used = torch.arange(tables.shape[1], device="cuda"), ((lens + page - 1) // page).view(-1, 1, 1)
    score = score.masked_fill(at >= used, -math.inf).masked_fill(at == used - 1, math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    best = torch.sort(best.masked_fill(best >= used, tables.shape[1]), dim=-1).values
    chosen = torch.full((B, hkv, top), -1, dtype=torch.int32, device="cuda")
    chosen[..., : best.shape[-1]] = best.masked_fill(best == tables.shape[1], -1)
    pages = tables.gather(1, chosen.clamp(min=0).long().view(B, -1)).view(B, hkv, top)
    heads = torch.arange(hkv, device="cuda").view(1, -1, 1)
    k, v = (t[pages, heads].float().flatten(2, 3) for t in (s["k_pages"], s["v_pages"]))  # [B, hkv, top * page, d]
    place = chosen.unsqueeze(-1) * page + torch.arange(page, device="cuda")
    has = ((chosen.unsqueeze(-1) >= 0) & (place < lens.view(-1, 1, 1, 1))).flatten(2, 3).unsqueeze(2)
    x = s["q"].float().view(B, hkv, G, d) @ k.transpose(2, 3).contiguous()
    p, total = _softmax(x.masked_fill(~has, -math.inf) * s["scale"])
    o = p @ v.masked_fill(~has.transpose(2, 3), 0.0) / total
    return o.reshape(B, hkv * G, d).to(s["q"].dtype), chosen


def _plain(s):
    op = s["case"]["op"]
    if op == "copy":
        src, dst = torch.tensor(s["src"], device="cuda"), torch.tensor(s["dst"], device="cuda")
        for_all = (s["k_pages"], s["v_pages"], s["bounds"])
        return [t.index_copy_(1, dst, t[:, src]) for t in for_all]
    return {"load": _plain_load, "store": _plain_store, "append": _plain_append, "shared": _plain_shared, "sparse": _plain_sparse}[op](s)


def run(s):
    if not own:
        return _plain(s)
    from megaqwen_amd import paged

    op = s["case"]["op"]
    if op == "copy":
        paged.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"], bounds=s["bounds"])
        return s["k_pages"], s["v_pages"], s["bounds"]
    if op == "load":
        paged.load_pages(s["k_cache"], s["v_cache"], s["k_pages"], s["v_pages"], s["pages"], s["case"]["n"], bounds=s["bounds"])
        return s["k_pages"], s["v_pages"], s["bounds"]
    if op == "store":
        paged.store_pages(s["k_pages"], s["v_pages"], s["pages"], s["case"]["n"], s["k_cache"], s["v_cache"])
        return s["k_cache"], s["v_cache"]
    if op == "append":
        paged.append_rows(s["k"], s["v"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], bounds=s["bounds"])
        return s["k_pages"], s["v_pages"], s["bounds"]
    if op == "shared":
        return paged.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix_pages"], s["prefix_len"], s["tables"],
                                             s["lens"], scale=s["scale"])
    return paged.sparse_attention(s["q"], s["k_pages"], s["v_pages"], s["bounds"], s["tables"], s["lens"], s["case"]["top"],
                                  scale=s["scale"])


def work(case):
    hkv, d, page = case["hkv"], case["d"], case["page"]
    row = 2 * hkv * d * 2  # one position's K and V rows of one layer
    if case["op"] == "copy":
        return {"bytes": 2 * case["n"] * case["layers"] * (page * row + 2 * hkv * d * 2), "flops": 0}
    if case["op"] in ("load", "store"):
        bounds = _pages(case["n"], page) * 2 * hkv * d * 2 if case["op"] == "load" else 0
        return {"bytes": case["layers"] * (2 * case["n"] * row + bounds), "flops": 0}
    lens, B = _lens(case), case["batch"]
    if case["op"] == "append":  # a row read and written, its page's bounds read and written
        return {"bytes": B * (2 * row + 2 * 2 * hkv * d * 2 + 8), "flops": 0}
    io = 2 * B * hkv * case["g"] * d * 2
    if case["op"] == "shared":
        n = case["prefix"]
        return {"bytes": io + (n + sum(lens)) * row + 4 * (_pages(n, page) + sum(_pages(x, page) for x in lens) + B),
                "flops": 4 * hkv * case["g"] * d * (B * n + sum(lens))}
    used = [_pages(x, page) for x in lens]
    read = [x if u <= case["top"] else (case["top"] - 1) * page + (x - 1) % page + 1 for x, u in zip(lens, used)]
    return {"bytes": io + sum(read) * row + sum(used) * (2 * hkv * d * 2 + 4) + 4 * B * (1 + hkv * case["top"]),
            "flops": 4 * hkv * case["g"] * d * (sum(read) + sum(used))}


def _exact_attend(q, k, v, scale):
    """q [h, d], k and v [rows, d] (one kv head's): softmax(q k^T scale) v in 64 bits; zeros without rows."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    x = (q @ k.t().contiguous()) * scale
    return torch.softmax(x, -1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "copy":
        out = [s[t].clone() for t in ("k_pages", "v_pages", "bounds")]
        for a, b in zip(s["src"], s["dst"]):
            for t, name in zip(out, ("k_pages", "v_pages", "bounds")):
                t[:, b] = s[name][:, a]
        return out
    if case["op"] in ("load", "store"):
        for i, p in enumerate(s["pages"]):
            lo, n = i * page, min(page, case["n"] - i * page)
            for pool, cache in (("k_pages", "k_cache"), ("v_pages", "v_cache")):
                inside, flat = s[pool][:, p, :, :n], s[cache][:, :, lo: lo + n]
                inside.copy_(flat) if case["op"] == "load" else flat.copy_(inside)
            keys = s["k_pages"][:, p, :, :n].double()
            s["bounds"][:, p, :, 0], s["bounds"][:, p, :, 1] = keys.amin(2), keys.amax(2)
        return (s["k_pages"], s["v_pages"], s["bounds"]) if case["op"] == "load" else (s["k_cache"], s["v_cache"])
    tables, lens = s["tables"].tolist(), s["lens"].tolist()
    if case["op"] == "append":
        for b, n in enumerate(lens):
            p, i = tables[b][n // page], n % page
            s["k_pages"][p, :, i], s["v_pages"][p, :, i] = s["k"][b], s["v"][b]
            seen = s["k"][b].double().unsqueeze(1)
            if i > 0:
                seen = torch.cat((s["bounds"][p].double(), seen), 1)
            s["bounds"][p, :, 0], s["bounds"][p, :, 1] = seen.amin(1), seen.amax(1)
        return s["k_pages"], s["v_pages"], s["bounds"]
    G, out = case["g"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    shared = s["prefix_pages"].tolist() if case["op"] == "shared" else []
    full = case.get("prefix", 0)
    pool_k, pool_v = s["k_pages"], s["v_pages"]
    chosen = torch.full((case["batch"], case["hkv"], case.get("top", 1)), -1, dtype=torch.int32)
    before = [[t[shared, j].reshape(-1, case["d"])[:full].double() for t in (pool_k, pool_v)] for j in range(case["hkv"])] if shared else None
    for b, n in enumerate(lens):
        mine = tables[b][: _pages(n, page)]
        for j in range(case["hkv"]):
            q = s["q"][b, j * G: (j + 1) * G].double()
            use = list(range(len(mine)))
            if case["op"] == "sparse":
                lo, hi = s["bounds"][mine, j].double().unbind(1)
                score = (q.clamp(min=0) @ hi.t().contiguous() + q.clamp(max=0) @ lo.t().contiguous()).sum(0).tolist()
                score[-1] = math.inf
                use = sorted(sorted(use, key=lambda i: (-score[i], i))[: case["top"]])
                chosen[b, j, : len(use)] = torch.tensor(use, dtype=torch.int32)
            kept = torch.tensor([i * page + r for i in use for r in range(min(page, n - i * page))], dtype=torch.long, device="cuda")
            ids = torch.tensor(mine, dtype=torch.long, device="cuda")
            k, v = (t[ids, j].reshape(-1, case["d"])[kept].double() if n else t.new_zeros(0, case["d"], dtype=torch.float64) for t in (pool_k, pool_v))
            if before:
                k, v = torch.cat((before[j][0], k)), torch.cat((before[j][1], v))
            out[b, j * G: (j + 1) * G] = _exact_attend(q, k, v, s["scale"])
    return out if case["op"] == "shared" else (out, chosen.cuda())
