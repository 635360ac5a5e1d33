"""A paged K/V cache for sequences that share rows, and the attentions that read it.

The decoders of `megakernel_decode` keep one contiguous cache each, as the reference does
(`csrc/megakernel/megakernel_decode.py:140-146`; it has no counterpart of this module). Here K and V rows
live in pages of a pool, `[layers, pages, kv heads, page size, head dim]`, and a sequence is a list
of page ids, so that sequences that begin alike (several answers to one prompt) share pages.

The functions work on tensors: `copy_pages`, `load_pages`, `store_pages` and `append_rows` move rows,
`shared_prefix_attention` and `sparse_attention` read them. `PagedKVCache` keeps the books for them:
which pages are free, which sequence uses which, and which have to be copied before a sequence
writes to them. All launches go to torch's current stream of the tensors' device; none
waits for the device or copies from host memory, and all can be captured into a HIP graph.

Types: bfloat16 and float16. Page sizes: 16, 32, 64, 128, 256. Head dims: 64 and 128. There is
no CPU fallback: tensors are on the GPU. Wrong types, shapes, strides or page ids raise ValueError.
"""

from __future__ import annotations

import ctypes
import functools
import heapq
import math

import torch

from . import _abi
from .config import HEAD_DIM, NUM_KV_HEADS, NUM_LAYERS

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
_DTYPES = {torch.bfloat16: _abi.MQ_BF16, torch.float16: _abi.MQ_FP16}


def _call(name: str, device: torch.device, *args) -> None:
    """C ABI entry `name` with `args` and the current stream of `device`, on that device."""
    if device.type != "cuda":
        raise ValueError(f"expected tensors on the GPU, got {device}")
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _call(name, device, *args)
    status = getattr(_abi.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if status:
        _abi.check(status, name)


def _like(t, name: str, dtype, device, shape=None) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or (shape is not None and t.shape != shape):
        got = (t.dtype, list(t.shape), str(t.device)) if isinstance(t, torch.Tensor) else t
        raise ValueError(f"{name}: expected {dtype} {'' if shape is None else list(shape)} on {device}, got {got}")


def _pool(k_pages, v_pages, bounds, layered: bool) -> _abi.MqPagePool:
    """The pool's descriptor, after its checks. layered: [layers, ...], else one layer's [pages, ...]."""
    dims = 5 if layered else 4
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != dims or k_pages.dtype not in _DTYPES:
        raise ValueError(f"k_pages: expected a tensor of {dims} dimensions, bfloat16 or float16")
    shape, dtype, device = k_pages.shape, k_pages.dtype, k_pages.device
    _like(v_pages, "v_pages", dtype, device, shape)
    layers, pages, heads, page, d = shape if layered else (1, *shape)
    if page not in PAGE_SIZES or d not in HEAD_DIMS or pages == 0 or heads == 0 or layers == 0:
        raise ValueError(f"k_pages: page size {page} (of {PAGE_SIZES}) or head dim {d} (of {HEAD_DIMS}) or a size of zero")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages, v_pages: expected contiguous tensors")
    at = None
    if bounds is not None:
        _like(bounds, "bounds", dtype, device, (layers, pages, heads, 2, d) if layered else (pages, heads, 2, d))
        if not bounds.is_contiguous():
            raise ValueError("bounds: expected a contiguous tensor")
        at = bounds.data_ptr()
    return _abi.MqPagePool(k_pages.data_ptr(), v_pages.data_ptr(), at, layers, pages, heads, page, d, _DTYPES[dtype])


def _page_list(ids, name: str, num_pages: int):
    """A host list of page ids, and as a C array."""
    ids = [int(i) for i in ids]
    if ids and (min(ids) < 0 or max(ids) >= num_pages):
        raise ValueError(f"{name}: page ids must be in [0, {num_pages})")
    return ids, (ctypes.c_int * len(ids))(*ids)


def copy_pages(k_pages, v_pages, src, dst, bounds=None) -> None:
    """Page `dst[i]` = page `src[i]` of every layer, K and V (and bounds). `src` and `dst` are host lists
    of the same length; the pages in `dst` differ from each other and from all in `src`."""
    pool = _pool(k_pages, v_pages, bounds, True)
    src, c_src = _page_list(src, "src", pool.num_pages)
    dst, c_dst = _page_list(dst, "dst", pool.num_pages)
    if not (len(src) == len(dst)):
        raise ValueError("src and dst: expected lists of one length")
    if not (len(set(dst)) == len(dst) and not set(dst) & set(src)):
        raise ValueError("dst: a page twice, or one that is copied from as well")
    if src:
        _call("mq_pages_copy", k_pages.device, pool, c_src, c_dst, len(src))


def _move(name, k_cache, v_cache, k_pages, v_pages, pages, length, bounds) -> None:
    pool = _pool(k_pages, v_pages, bounds, True)
    pages, c_pages = _page_list(pages, "pages", pool.num_pages)
    length = int(length)
    if not (length >= 0 and len(pages) == -(-length // pool.page_size)):
        raise ValueError(f"pages: {length} rows need {-(-length // pool.page_size)} pages of {pool.page_size}, got {len(pages)}")
    if len(set(pages)) != len(pages):
        raise ValueError("pages: a page twice")
    if not (isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4):
        raise ValueError("k_cache: expected [layers, kv heads, positions, head dim]")
    shape = (pool.num_layers, pool.num_kv_heads, k_cache.shape[2], pool.head_dim)
    for t, what in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _like(t, what, k_pages.dtype, k_pages.device, shape)
        if not t.is_contiguous():
            raise ValueError(f"{what}: expected a contiguous tensor")
    if length > shape[2]:
        raise ValueError(f"length {length} exceeds the cache's {shape[2]} positions")
    if length:
        _call(name, k_pages.device, pool, c_pages, length, k_cache.data_ptr(), v_cache.data_ptr(), shape[2])


def load_pages(k_cache, v_cache, k_pages, v_pages, pages, length: int, bounds=None) -> None:
    """Positions 0 .. length - 1 of a decoder's contiguous caches `[layers, kv heads, positions, head
    dim]` into the pages of the host list `pages`, and with `bounds` those pages' bounds. Rows behind
    `length` in the last page stay as they are."""
    _move("mq_pages_load", k_cache, v_cache, k_pages, v_pages, pages, length, bounds)


def store_pages(k_pages, v_pages, pages, length: int, k_cache, v_cache) -> None:
    """The inverse of `load_pages`: the first `length` rows of `pages` into contiguous caches, whose
    other positions stay as they are."""
    _move("mq_pages_store", k_cache, v_cache, k_pages, v_pages, pages, length, None)


def _rows(t, name: str, dtype, device, shape) -> tuple[int, int]:
    """(batch, head) strides in elements of a [batch, heads, d] tensor of the pool's type."""
    _like(t, name, dtype, device, shape)
    sb, sh, sd = t.stride()
    # (a stride over one element is never used, whatever it says)
    if shape[0] == 1:
        sb = 0
    if shape[1] == 1:
        sh = 0
    if not (sd == 1 and sb >= 0 and sh >= 0 and (sb | sh) & 7 == 0 and t.data_ptr() & 15 == 0):
        raise ValueError(f"{name}: expected rows of contiguous elements that begin at multiples of 16 bytes, got strides {t.stride()}")
    return sb, sh


def _tables(tables, lens, batch: int, device) -> tuple[int, int]:
    """(row stride, width) of int32 page tables [batch, width]."""
    n, width = tables.shape if isinstance(tables, torch.Tensor) and tables.dim() == 2 else (0, 0)
    if n != batch or not 1 <= width <= _abi.MQ_MAX_TABLE_WIDTH:
        raise ValueError(f"tables: expected int32 [{batch}, 1 .. {_abi.MQ_MAX_TABLE_WIDTH}]")
    _like(tables, "tables", torch.int32, device)
    _like(lens, "lens", torch.int32, device, (batch,))
    row, entry = tables.stride()
    if (width > 1 and entry != 1) or (batch > 1 and (row < 0 or lens.stride(0) != 1)):
        raise ValueError("tables, lens: expected contiguous rows")
    return (row if batch > 1 else 0), width


def append_rows(k, v, k_pages, v_pages, tables, lens, bounds=None) -> None:
    """One new K and V row a sequence, `k` and `v` `[batch, kv heads, head dim]`, to position `lens[b]` of the
    sequence with page table `tables[b]`, in one layer's `[pages, kv heads, page size, head dim]`, and
    with `bounds` the page's bounds. `lens` itself does not change. No two sequences may append to
    one page; a row for a position behind its table, or for a page outside the pool, is dropped."""
    pool = _pool(k_pages, v_pages, bounds, False)
    if not (isinstance(k, torch.Tensor) and k.dim() == 3 and 1 <= k.shape[0] <= 65535):
        raise ValueError("k: expected [batch, kv heads, head dim]")
    batch, dtype, device = k.shape[0], k_pages.dtype, k_pages.device
    shape = (batch, pool.num_kv_heads, pool.head_dim)
    k_sb, k_sh = _rows(k, "k", dtype, device, shape)
    v_sb, v_sh = _rows(v, "v", dtype, device, shape)
    t_sb, width = _tables(tables, lens, batch, device)
    _call("mq_pages_append", device, pool, k.data_ptr(), v.data_ptr(), k_sb, k_sh, v_sb, v_sh, tables.data_ptr(), t_sb, width,
          lens.data_ptr(), batch)


def _query(q, out, pool, dtype, device):
    """(shape, out, q's (batch, head) strides, out's) of an attention call."""
    shape = tuple(q.shape) if isinstance(q, torch.Tensor) else ()
    if not (len(shape) == 3 and 1 <= shape[0] <= 65535 and 0 < shape[1] <= 16384 and shape[1] % pool.num_kv_heads == 0
            and shape[2] == pool.head_dim):
        raise ValueError(f"q: expected [batch, a multiple of {pool.num_kv_heads} heads, {pool.head_dim}]")
    strides = _rows(q, "q", dtype, device, shape)
    if out is None:
        out = torch.empty_like(q)
        sb, sh, _ = out.stride()
        return shape, out, strides, (sb if shape[0] > 1 else 0, sh if shape[1] > 1 else 0)
    out_strides = _rows(out, "out", dtype, device, shape)
    span = shape[2]
    for stride, n in sorted(zip(out_strides, shape)):
        if n > 1 and stride < span:
            raise ValueError(f"out: rows that overlap, strides {out.stride()}")
        span += stride * (n - 1)
    return shape, out, strides, out_strides


def _scale(scale, head_dim: int) -> float:
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    return scale


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(kv_heads: int, head_dim: int, heads: int, batch: int, prefix_len: int, max_len: int, top: int) -> int:
    n, pool = ctypes.c_size_t(), _abi.MqPagePool(num_kv_heads=kv_heads, head_dim=head_dim)
    _abi.check(_abi.lib().mq_attention_workspace(pool, heads, batch, prefix_len, max_len, top, n), "mq_attention_workspace")
    return n.value


def shared_prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len: int, tables, lens, scale: float | None = None,
                            max_len: int | None = None, out=None) -> torch.Tensor:
    """Attention of one query token a sequence, `q` `[batch, query heads, head dim]`, over a prefix that all
    sequences share and the sequence's own rows behind it: softmax(scale q K^T) V with K, V = prefix
    rows 0 .. prefix_len - 1, then own rows 0 .. lens[b] - 1. The prefix is read once for all sequences
    (for each 128 query rows of a kv head).

    One layer's pool; `prefix_pages` int32 on the GPU, `prefix_len` a host number (0: no prefix);
    `tables` int32 `[batch, width]` (rows may be a slice of wider ones), `lens` int32 `[batch]`. A sequence
    without any row gets zeros; one that needs a page outside the pool gets NaN. `max_len`: the longest of
    `lens`, if the caller knows it (default width * page size): it decides how the work is split, not what is
    computed. `scale` defaults to 1 / sqrt(head dim)."""
    pool = _pool(k_pages, v_pages, None, False)
    device = k_pages.device
    (batch, heads, d), out, (q_sb, q_sh), (o_sb, o_sh) = _query(q, out, pool, k_pages.dtype, device)
    t_sb, width = _tables(tables, lens, batch, device)
    prefix_len = int(prefix_len)
    if prefix_len < 0:
        raise ValueError("prefix_len must not be negative")
    if prefix_len:
        _like(prefix_pages, "prefix_pages", torch.int32, device)
        if not (prefix_pages.dim() == 1 and prefix_pages.is_contiguous()
                and prefix_pages.numel() >= -(-prefix_len // pool.page_size)):
            raise ValueError(f"prefix_pages: expected at least {-(-prefix_len // pool.page_size)} contiguous page ids")
    whole = width * pool.page_size
    max_len = whole if max_len is None else min(int(max_len), whole)
    if max_len < 1:
        raise ValueError("max_len must be positive")
    ws_bytes = _workspace_bytes(pool.num_kv_heads, d, heads, batch, prefix_len, max_len, 0)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    _call("mq_shared_prefix_attention", device, pool, q.data_ptr(), q_sb, q_sh, out.data_ptr(), o_sb, o_sh, heads, batch,
          prefix_pages.data_ptr() if prefix_len else None, prefix_len, tables.data_ptr(), t_sb, width, lens.data_ptr(), max_len,
          _scale(scale, d), ws.data_ptr() if ws_bytes else None, ws_bytes)
    return out


def sparse_attention(q, k_pages, v_pages, bounds, tables, lens, top_pages: int, scale: float | None = None,
                     out=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of one query token a sequence over `top_pages` of its pages: the last one and the others
    with the largest scores; all of them if there are no more. A page's score for a kv head is the sum,
    over the head's queries and the dims, of max(q lo, q hi), with `bounds` `[pages, kv heads, 2, head
    dim]` the least and greatest key entries (lo, hi) of the page: the most that the products with any key
    inside could add up to. It is summed in 64 bits; of equal scores the earlier page wins.

    Returns (out, chosen): `chosen` int32 `[batch, kv heads, top_pages]`, the pages' numbers in the
    sequence's table, ascending, then -1. The rest as `shared_prefix_attention` without a prefix."""
    if bounds is None:
        raise ValueError("bounds: expected a tensor")
    pool = _pool(k_pages, v_pages, bounds, False)
    device, top = k_pages.device, int(top_pages)
    (batch, heads, d), out, (q_sb, q_sh), (o_sb, o_sh) = _query(q, out, pool, k_pages.dtype, device)
    t_sb, width = _tables(tables, lens, batch, device)
    if not 1 <= top <= _abi.MQ_MAX_TABLE_WIDTH:
        raise ValueError(f"top_pages must be in [1, {_abi.MQ_MAX_TABLE_WIDTH}]")
    chosen = torch.empty(batch, pool.num_kv_heads, top, dtype=torch.int32, device=device)
    ws_bytes = _workspace_bytes(pool.num_kv_heads, d, heads, batch, 0, min(top, width) * pool.page_size, top)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    _call("mq_sparse_attention", device, pool, q.data_ptr(), q_sb, q_sh, out.data_ptr(), o_sb, o_sh, chosen.data_ptr(), heads,
          batch, tables.data_ptr(), t_sb, width, lens.data_ptr(), top, _scale(scale, d), ws.data_ptr(), ws_bytes)
    return out, chosen


class PagedKVCache:
    """The books of a page pool: sequences as lists of pages, shared until one of them writes.

    Sequences are numbers that `new`, `fork` and `free` hand out and take back. `fork` copies nothing: the
    new sequences use the same pages, and `reserve` gives a sequence a page of its own (a copy of the
    last one, if it is shared and not full) before a row is appended. `compact` moves the pages in
    use to the front of the pool.

    `k_pages`, `v_pages` `[layers, pages, kv heads, page size, head dim]` and, with `bounds=True`, `bounds`
    (for `sparse_attention`) are the pool; the functions of this module take them, or one layer of
    them. Rows that were appended by `append_rows` are made known with `extend`. A pool without a free
    page raises MegakernelError, before anything has changed."""

    def __init__(self, num_pages: int, num_layers: int = NUM_LAYERS, num_kv_heads: int = NUM_KV_HEADS, head_dim: int = HEAD_DIM,
                 page_size: int = 64, dtype=torch.bfloat16, device="cuda", bounds: bool = False):
        if dtype not in _DTYPES:
            raise ValueError(f"dtype: expected bfloat16 or float16, got {dtype}")
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page size {page_size} (of {PAGE_SIZES}) or head dim {head_dim} (of {HEAD_DIMS})")
        if min(num_pages, num_layers, num_kv_heads) < 1:
            raise ValueError("num_pages, num_layers and num_kv_heads must be positive")
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.page_size, self.num_pages = page_size, num_pages
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.bounds = torch.zeros(shape[:3] + (2, head_dim), dtype=dtype, device=device) if bounds else None
        self._free = list(range(num_pages))  # a heap: the lowest page first
        self._users = [0] * num_pages
        self._seqs: dict[int, list] = {}  # sequence -> [pages, rows]
        self._next = 0
        self.version = 0  # changes with every change of a page list or a length

    # -- the books ---------------------------------------------------------------
    def _of(self, seq: int) -> list:
        try:
            return self._seqs[seq]
        except KeyError:
            raise ValueError(f"no sequence {seq}") from None

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise _abi.MegakernelError(f"page pool exhausted: {n} pages wanted, {len(self._free)} of {self.num_pages} free")
        pages = [heapq.heappop(self._free) for _ in range(n)]
        for p in pages:
            self._users[p] = 1
        return pages

    def _drop(self, pages) -> None:
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                heapq.heappush(self._free, p)

    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, seq: int) -> list[int]:
        return list(self._of(seq)[0])

    def length(self, seq: int) -> int:
        return self._of(seq)[1]

    def new(self) -> int:
        """A sequence without rows."""
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = [[], 0]
        return seq

    def fork(self, seq: int, n: int = 1) -> list[int]:
        """n sequences with the rows of `seq`, whose pages they share. No row is copied. (Pages that were reserved
        and hold no row yet stay `seq`'s alone.)"""
        pages, rows = self._of(seq)
        if n < 0:
            raise ValueError("n must not be negative")
        pages = pages[: -(-rows // self.page_size)]
        out = []
        for _ in range(n):
            s = self.new()
            self._seqs[s] = [list(pages), rows]
            out.append(s)
        for p in pages:
            self._users[p] += n
        return out

    def free(self, seq: int) -> None:
        """Gives the sequence's pages back, those that no other sequence uses to the pool."""
        pages, _ = self._of(seq)
        del self._seqs[seq]
        self._drop(pages)
        self.version += 1

    def reserve(self, seqs, rows: int = 1) -> None:
        """Makes room for `rows` more rows behind each sequence: new pages, and a copy of a last page that
        others use too and that is not full (one launch for all of them)."""
        if rows < 0:
            raise ValueError("rows must not be negative")
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("seqs: a sequence twice")
        users, plan, want = {}, [], 0
        for s in seqs:
            pages, n = self._of(s)
            more = max(0, -(-(n + rows) // self.page_size) - len(pages))
            own = False
            if rows and n % self.page_size:
                last = pages[n // self.page_size]
                left = users.get(last, self._users[last])
                own = left > 1
                users[last] = left - own
            plan.append((pages, n, more, own))
            want += more + own
        if not want:
            return
        taken = iter(self._take(want))
        src, dst = [], []
        for pages, n, more, own in plan:
            if own:
                at = n // self.page_size
                src.append(pages[at])
                dst.append(next(taken))
                self._users[pages[at]] -= 1
                pages[at] = dst[-1]
            pages.extend(next(taken) for _ in range(more))
        self.version += 1
        if src:
            copy_pages(self.k_pages, self.v_pages, src, dst, bounds=self.bounds)

    def extend(self, seqs, rows: int = 1) -> None:
        """`rows` rows were appended to each sequence (within what `reserve` made room for)."""
        seqs = list(seqs)
        for s in seqs:
            pages, n = self._of(s)
            if not 0 <= n + rows <= len(pages) * self.page_size or rows < 0:
                raise ValueError(f"sequence {s}: {n} + {rows} rows do not fit its {len(pages)} pages")
        for s in seqs:
            self._seqs[s][1] += rows
        self.version += 1

    def load(self, seq: int, k_cache, v_cache, length: int) -> None:
        """Rows 0 .. length - 1 of contiguous caches as all of the sequence's rows (it has none yet)."""
        pages, n = self._of(seq)
        if pages or n:
            raise ValueError(f"sequence {seq} has rows already")
        if length < 0:
            raise ValueError("length must not be negative")
        taken = self._take(-(-length // self.page_size))
        try:
            load_pages(k_cache, v_cache, self.k_pages, self.v_pages, taken, length, bounds=self.bounds)
        except BaseException:
            self._drop(taken)
            raise
        self._seqs[seq] = [taken, length]
        self.version += 1

    def store(self, seq: int, k_cache, v_cache) -> int:
        """The sequence's rows into contiguous caches, from position 0; returns how many."""
        pages, n = self._of(seq)
        store_pages(self.k_pages, self.v_pages, pages[: -(-n // self.page_size)], n, k_cache, v_cache)
        return n

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool, one launch; returns their number. Page lists are
        rewritten; tables made before are void."""
        used = [p for p, u in enumerate(self._users) if u]
        src = [p for p in used if p >= len(used)]
        if not src:
            return len(used)
        dst = [p for p in range(len(used)) if not self._users[p]]
        copy_pages(self.k_pages, self.v_pages, src, dst, bounds=self.bounds)
        to = dict(zip(src, dst))
        for entry in self._seqs.values():
            entry[0] = [to.get(p, p) for p in entry[0]]
        for a, b in to.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(len(used), self.num_pages))
        self.version += 1
        return len(used)

    # -- what the attentions read --------------------------------------------------
    def shared_pages(self, seqs) -> int:
        """How many pages all of the sequences begin with, full in every one of them."""
        lists = [self._of(s) for s in seqs]
        if not lists:
            return 0
        most = min(n for _, n in lists) // self.page_size
        first = lists[0][0]
        for at in range(most):
            if any(pages[at] != first[at] for pages, _ in lists):
                return at
        return most

    def tables(self, seqs, first: int = 0):
        """(tables, lens) of the sequences on the GPU, int32 `[n, width]` and `[n]`, from their page number `first` on:
        all pages they have, room that was reserved included, and the rows in them so far."""
        lists = [self._of(s) for s in seqs]
        if not lists:
            raise ValueError("seqs: expected at least one sequence")
        width = max(1, max(len(pages) - first for pages, _ in lists))
        if width > _abi.MQ_MAX_TABLE_WIDTH:
            raise ValueError(f"a sequence of {width} pages exceeds the table width {_abi.MQ_MAX_TABLE_WIDTH}")
        table = [pages[first:] + [-1] * (width - max(0, len(pages) - first)) for pages, _ in lists]
        lens = [max(0, n - first * self.page_size) for _, n in lists]
        device = self.k_pages.device
        return torch.tensor(table, dtype=torch.int32).to(device), torch.tensor(lens, dtype=torch.int32).to(device)
