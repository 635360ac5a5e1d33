"""GPU tests of decoding several sequences at once (MegakernelBatchDecoder, mq_decode_batch) against the
batch-1 decoder on the same contexts.

The two run the same products in the same order and differ in the order of the attention's sums, so their
logits agree within the tolerances that the kernels' own parity tests use for such
differences (parity_helpers: LOGIT_MAX_ABS, LOGIT_MEAN_ABS), and greedy tokens agree outside near-ties."""

import ctypes

import pytest
import torch

from megaqwen_amd import _abi, paged, rope, weights
from megaqwen_amd import megakernel_decode as MK
from parity_helpers import LOGIT_MAX_ABS, LOGIT_MEAN_ABS, TIE_TOL

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small(state_dict):
    """A 2-layer decoder and one more like it for the expected results."""
    flat = [t.cuda() for t in weights.layer_weights_flat(state_dict, 2)]
    embed, norm = state_dict["model.embed_tokens.weight"].cuda(), state_dict["model.norm.weight"].cuda()
    cos, sin = (t.cuda() for t in rope.rope_tables(1024))
    return [MK.MegakernelPrefillDecoder(embed, flat, norm, embed, cos, sin, 2, 1024, max_prefill_len=1000) for _ in range(2)]


def _close(got, want, tok=None):
    d = (got - want).abs()
    assert float(d.max()) <= LOGIT_MAX_ABS and float(d.mean()) <= LOGIT_MEAN_ABS, (float(d.max()), float(d.mean()))
    if tok is not None:
        assert int(got.argmax()) == tok
        top = torch.topk(want, 2).values
        if float(top[0] - top[1]) > TIE_TOL:
            assert tok == int(want.argmax())


def _expect(single, ids):
    """(token, logits) of the batch-1 decoder behind the context ids[:-1] for the token ids[-1]."""
    single.reset()
    if len(ids) > 1:
        single.prefill_step(ids[:-1])
    return single.decode_step_with_logits(ids[-1])


@pytest.mark.parametrize("page", [16, 64, 256])
def test_forks_of_one_prompt(small, page):
    """Prompt, three forks, forced tokens that part at the first step; every step of every fork."""
    dec, single = small
    prompt = weights.random_prompt(150, seed=page)
    b = MK.MegakernelBatchDecoder(dec, max_batch=4, page_size=page, num_pages=80)
    seq, tok = b.prefill(prompt)
    single.reset()
    assert tok == single.prefill_step(prompt)
    seqs = [seq] + b.fork(seq, 3)
    rows = [list(prompt) for _ in seqs]
    forced = [weights.random_prompt(4, seed=900 + i) for i in range(5)]
    for step in range(5):
        for r, t in zip(rows, forced[step]):
            r.append(t)
        toks, logits = b.step_with_logits(seqs, forced[step])
        for i, r in enumerate(rows):
            _close(logits[i], _expect(single, r)[1], toks[i])
        assert [b.length(s) for s in seqs] == [len(r) for r in rows]
    # the rows that the steps appended, handed back to the batch-1 decoder
    b.to_decoder(seqs[2])
    assert dec.position() == len(rows[2])
    n = len(prompt)
    _expect(single, rows[2] + [1])
    a, w = dec.get_k_cache()[:, :, :n + 5].float(), single.get_k_cache()[:, :, :n + 5].float()
    assert torch.equal(a[:, :, :n], w[:, :, :n])  # (the same prefill)
    assert float((a - w).norm() / w.norm()) < 1e-2
    tok, lg = dec.decode_step_with_logits(77)
    _close(lg, _expect(single, rows[2] + [77])[1], tok)


def test_sequences_without_a_common_prefix(small):
    """Prompts of other lengths (one empty, one of a token), in an order of their own, joined and left."""
    dec, single = small
    b = MK.MegakernelBatchDecoder(dec, max_batch=8, page_size=32, num_pages=100)
    rows = [weights.random_prompt(n, seed=n + 1) for n in (31, 0, 300, 1, 64)]
    seqs = [b.prefill(r)[0] if r else b.new() for r in rows]
    for step, order in enumerate(([0, 1, 2, 3, 4], [4, 2, 0], [1], [3, 1, 4, 0, 2])):
        toks = weights.random_prompt(len(order), seed=50 + step)
        got, logits = b.step_with_logits([seqs[i] for i in order], toks)
        for j, i in enumerate(order):
            rows[i] = list(rows[i]) + [toks[j]]
            _close(logits[j], _expect(single, rows[i])[1], got[j])
    for s in seqs:
        b.free(s)
    assert b.cache.free_pages() == 100


@pytest.mark.parametrize("n", [1, 2, 33, 64, 65, 130, 300, 520])
def test_batch_sizes(small, n):
    """Every shape of the products and of the shared prefix's tiles: equal sequences give equal rows."""
    dec, single = small
    prompt = weights.random_prompt(200, seed=n)
    b = MK.MegakernelBatchDecoder(dec, max_batch=n, page_size=64, num_pages=3 + 2 * n)
    root, _ = b.prefill(prompt)
    seqs = b.fork(root, n)
    b.free(root)
    print(f"batch {n}", flush=True)
    _, want = _expect(single, prompt + [5])
    toks, logits = b.step_with_logits(seqs, [5] * n)
    _close(logits[0], want, toks[0])
    assert toks == [toks[0]] * n and all(torch.equal(logits[i], logits[0]) for i in range(n))
    toks, logits = b.step_with_logits(seqs, [9] * n)
    _close(logits[n - 1], _expect(single, prompt + [5, 9])[1], toks[n - 1])
    assert toks == [toks[0]] * n


def test_full_model_batch(gpu_weights):
    """All 28 layers: four continuations of a 400-token prompt, three forced steps."""
    w = dict(gpu_weights)
    mk = lambda: MK.MegakernelPrefillDecoder(w["embed_weight"], w["layer_weights"], w["final_norm_weight"], w["lm_head_weight"],  # noqa: E731
                                             w["cos_table"], w["sin_table"], 28, 1024, max_prefill_len=512)
    dec, single = mk(), mk()
    prompt = weights.random_prompt(400, seed=3)
    b = MK.MegakernelBatchDecoder(dec, max_batch=4, num_pages=20)
    seq, _ = b.prefill(prompt)
    seqs = [seq] + b.fork(seq, 3)
    rows = [list(prompt) for _ in seqs]
    for step in range(3):
        forced = weights.random_prompt(4, seed=70 + step)
        toks, logits = b.step_with_logits(seqs, forced)
        for i in range(4):
            rows[i].append(forced[i])
            _close(logits[i], _expect(single, rows[i])[1], toks[i])


def test_sparse_pages(small):
    """With room for every page the choice takes them all: bit-identical to no choice. With fewer, the step runs on
    the bounds that load, copies and appends keep up: they equal the pages' own."""
    dec, _ = small
    prompt = weights.random_prompt(700, seed=12)
    forced = weights.random_prompt(20, seed=13)
    results = []
    for top in (None, 64, 4):
        b = MK.MegakernelBatchDecoder(dec, max_batch=2, page_size=32, num_pages=60, sparse_pages=top)
        seq, _ = b.prefill(prompt)
        out = [b.step_with_logits([seq], [t])[1] for t in forced]
        results.append(torch.stack(out))
        if top == 4:
            other = b.fork(seq)[0]
            b.step([seq, other], [3, 4])
            cache = b.cache
            for s in (seq, other):
                for i, p in enumerate(cache.pages(s)):
                    rows = cache.k_pages[:, p, :, : min(32, cache.length(s) - 32 * i)]
                    assert torch.equal(cache.bounds[:, p], torch.stack((rows.amin(-2), rows.amax(-2)), -2))
    assert torch.equal(results[0], results[1])
    assert bool(results[2].isfinite().all()) and not torch.equal(results[0], results[2])


def test_rows_that_a_user_appends_between_steps(small):
    """The pool is the user's too: rows appended with append_rows and extend count in the next step of the same sequences."""
    dec, _ = small
    prompt = weights.random_prompt(100, seed=30)
    b = MK.MegakernelBatchDecoder(dec, max_batch=2, page_size=64, num_pages=20)
    seq, _ = b.prefill(prompt)
    one, two = b.fork(seq, 2)
    cache = b.cache
    b.step([one], [1])
    b.step([two], [1])
    cache.reserve([one])
    tables, lens = cache.tables([one])
    row = torch.randn(2, 1, 8, 128, device="cuda").to(torch.bfloat16)
    for l in range(2):
        paged.append_rows(row[l], row[l], cache.k_pages[l], cache.v_pages[l], tables, lens)
    cache.extend([one])
    got = b.step_with_logits([one], [7])[1]
    # the same rows by way of the batch-1 cache
    dec.reset()
    b.to_decoder(two)
    dec.k_cache_[:, :, 101], dec.v_cache_[:, :, 101] = row[:, 0], row[:, 0]
    dec.set_position(102)
    _close(got[0], dec.decode_step_with_logits(7)[1])


def test_a_step_that_is_cut_short_leaves_no_stale_lengths(small):
    """An error after the launch, which has advanced the lengths on the GPU: the next step starts from the books."""
    dec, single = small
    prompt = weights.random_prompt(40, seed=31)
    b = MK.MegakernelBatchDecoder(dec, max_batch=2, page_size=16, num_pages=20)
    seqs = [b.prefill(prompt)[0]]
    seqs += b.fork(seqs[0])
    b.step(seqs, [1, 2])

    def cut(*_):
        raise KeyboardInterrupt

    b.cache.extend = cut
    with pytest.raises(KeyboardInterrupt):
        b.step(seqs, [3, 4])
    del b.cache.extend
    got, logits = b.step_with_logits(seqs, [5, 6])
    for i in range(2):
        _close(logits[i], _expect(single, list(prompt) + [1 + i, 5 + i])[1], got[i])


def test_step_refusals(small):
    dec, _ = small
    b = MK.MegakernelBatchDecoder(dec, max_batch=2, page_size=16, num_pages=3)
    s = b.prefill(weights.random_prompt(20, seed=1))[0]
    t = b.fork(s)[0]
    for seqs, toks in (([], []), ([s], [1, 2]), ([s, s], [1, 2]), ([s, t, s], [1, 2, 3]), ([99], [1]), ([s], [-1]), ([s], [151936])):
        with pytest.raises(ValueError):
            b.step(seqs, toks)
    b.step([s, t], [1, 2])  # takes the third page
    u = b.fork(s)[0]
    with pytest.raises(_abi.MegakernelError, match="exhausted"):
        b.step([s, u], [1, 2])
    assert b.length(s) == 21 and b.length(u) == 20 + 1
    b.free(t)
    b.step([s, u], [1, 2])
    for bad in (dict(max_batch=0), dict(max_batch=1025), dict(page_size=20), dict(sparse_pages=0)):
        with pytest.raises(ValueError):
            MK.MegakernelBatchDecoder(dec, **{"max_batch": 1, "num_pages": 2, **bad})


def _raw_step(dec, pool, ids, lens, tables, prefix_pages, prefix_len, logits=None, ws=None, out=None):
    n, width = tables.shape
    size = ctypes.c_size_t()
    max_len = width * pool.page_size
    _abi.check(_abi.lib().mq_decode_batch_workspace(pool, n, prefix_len, max_len, 0, width, size), "workspace")
    ws = torch.empty(size.value, dtype=torch.uint8, device="cuda") if ws is None else ws
    out = torch.full((n,), -99, dtype=torch.int32, device="cuda") if out is None else out
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    st = _abi.lib().mq_decode_batch(p(ids), p(out), p(logits), n, p(dec.embed_weight_), ctypes.addressof(dec.h_layer_weights_),
                                    p(dec.final_norm_weight_), p(dec.lm_head_weight_), p(dec.cos_table_), p(dec.sin_table_),
                                    dec.cos_table_.shape[0], pool, p(prefix_pages), prefix_len, p(tables), width, width, p(lens),
                                    max_len, 0, dec.attn_scale_, p(ws), size.value, torch.cuda.current_stream().cuda_stream)
    assert st == _abi.MQ_OK
    return out, ws


def _int(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_step_reports_what_it_could_not_do(small):
    """Ids outside the vocabulary, positions outside the tables and missing pages: a negative token and an unchanged length,
    and the other sequences as if alone."""
    dec, _ = small
    cache = paged.PagedKVCache(8, 2, page_size=16)
    pool = paged._pool(cache.k_pages, cache.v_pages, None, True)
    good, _ = _raw_step(dec, pool, _int(11), _int(0), _int(0).view(1, 1), None, 0)
    ids = _int(11, -1, 151936, 11, 11, 11, 11)
    lens = _int(0, 0, 0, -3, 16, 0, 5000)
    tables = torch.tensor([[1], [2], [3], [4], [5], [-1], [6]], dtype=torch.int32, device="cuda")
    out, _ = _raw_step(dec, pool, ids, lens, tables, None, 0)
    assert out.tolist() == [int(good[0]), -2, -2, -3, -3, -5, -3]
    assert lens.tolist() == [1, 0, 0, -3, 16, 0, 5000]
    # behind a prefix the RoPE table ends earlier
    lens = _int(1, 15)
    out, _ = _raw_step(dec, pool, _int(11, 11), lens, _int(0, 1).view(2, 1), torch.arange(1009 // 16 + 1, dtype=torch.int32, device="cuda") % 8, 1009)
    assert out[0] >= 0 and int(out[1]) == -3 and lens.tolist() == [2, 15]


def test_step_in_a_captured_graph(small):
    """The step captured once and replayed, with eager steps between the replays: tokens, lengths and pages as by eager steps."""
    dec, _ = small
    prompt = weights.random_prompt(70, seed=21)
    results = []
    for captured in (False, True):
        cache = paged.PagedKVCache(12, 2, page_size=64)
        dec.reset()
        dec.prefill_step(prompt)
        a = cache.new()
        cache.load(a, dec.get_k_cache(), dec.get_v_cache(), 70)
        seqs = [a] + cache.fork(a, 2)
        cache.reserve(seqs, 8)
        tables, lens = cache.tables(seqs, 1)
        prefix = _int(*cache.pages(a)[:1])
        pool = paged._pool(cache.k_pages, cache.v_pages, None, True)
        ids, logits = _int(5, 6, 7), torch.empty(3, 151936, dtype=torch.bfloat16, device="cuda")
        out, ws = _raw_step(dec, pool, ids, lens, tables, prefix, 64, logits)
        torch.cuda.synchronize()
        seen = [(out.tolist(), logits.clone())]
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                _raw_step(dec, pool, ids, lens, tables, prefix, 64, logits, ws, out)
        for i in range(5):
            ids.copy_(out)
            if captured and i != 2:
                graph.replay()
            else:
                _raw_step(dec, pool, ids, lens, tables, prefix, 64, logits, ws, out)
            seen.append((out.tolist(), logits.clone()))
        assert lens.tolist() == [12, 12, 12]
        results.append((seen, cache.k_pages.clone(), cache.v_pages.clone()))
    for (ta, la), (tb, lb) in zip(results[0][0], results[1][0]):
        assert ta == tb and torch.equal(la, lb)
    assert torch.equal(results[0][1], results[1][1]) and torch.equal(results[0][2], results[1][2])


def test_generate_many(state_dict):
    """The generator's path: greedy copies, sampled ones that part and repeat with their seed, stop tokens, the cache limit."""
    flat = [t.cuda() for t in weights.layer_weights_flat(state_dict, 2)]
    embed = state_dict["model.embed_tokens.weight"].cuda()
    cos, sin = rope.rope_tables(128)
    w = {"embed_weight": embed, "layer_weights": flat, "final_norm_weight": state_dict["model.norm.weight"].cuda(),
         "lm_head_weight": embed, "cos_table": cos.cuda(), "sin_table": sin.cuda()}
    gen = MK.MegakernelPrefillGenerator(max_seq_len=128, max_prefill_len=100, weights_dict=w)
    prompt = weights.random_prompt(40, seed=5)
    many = gen.generate_many_ids(prompt, 3, max_new_tokens=10)
    assert many == [many[0]] * 3 and len(many[0]) == 10
    sampled = gen.generate_many_ids(prompt, 5, max_new_tokens=8, do_sample=True, temperature=2.0, seed=1)
    assert len({tuple(x) for x in sampled}) == 5 and all(len(x) == 8 for x in sampled)
    assert sampled == gen.generate_many_ids(prompt, 5, max_new_tokens=8, do_sample=True, temperature=2.0, seed=1)
    stop = sampled[2][3]
    cut = gen.generate_many_ids(prompt, 5, max_new_tokens=8, do_sample=True, temperature=2.0, seed=1, stop_tokens=[stop])
    assert all(stop not in x for x in cut) and cut[2] == sampled[2][:sampled[2].index(stop)]
    # (until the cache is full, as the single generator: the prompt's 40 tokens and 87 more, less the last step's)
    full = gen.generate_many_ids(prompt, 2, max_new_tokens=500)
    assert len(full[0]) == 128 - 1 - 39
    assert gen.generate_many_ids(prompt[:1], 2, max_new_tokens=3)[0] == gen.generate_many(prompt[:1], 1, max_new_tokens=3)[0]
    assert gen.generate_many_ids(prompt, 2, max_new_tokens=6, sparse_pages=2) == gen.generate_many_ids(prompt, 2, max_new_tokens=6)
    assert gen.batch_decoder_.cache.free_pages() == gen.batch_decoder_.cache.num_pages
    assert gen.generate_many_ids(prompt, 2, max_new_tokens=0) == [[], []]
    for bad in (dict(n=0), dict(n=1025), dict(n=1, do_sample=True, temperature=0.0)):
        with pytest.raises(ValueError):
            gen.generate_many_ids(prompt, **bad)
    with pytest.raises(ValueError):
        gen.generate_many_ids([], 2)
