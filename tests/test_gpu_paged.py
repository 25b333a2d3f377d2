"""The paged key-value cache (qc_paged_append, qc_paged_attention, qc_paged_evict) against plain 64-bit
forms.  Slots that no sequence has cached hold NaN throughout, so a read past a length shows."""
import math

import pytest
import torch

from _paged import DTYPE, Cache, attention64, evict64, ptr

pytestmark = pytest.mark.gpu


def run_attention(E, cache, q, seq, lens, lse=True, weights=None, scale=0.0, stream=None, out=None):
    rows, heads, D = q.shape
    sq = torch.tensor(seq, dtype=torch.int32, device="cuda") if seq is not None else None
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((rows, heads, D), 7.0, device="cuda") if out is None else out
    ls = torch.full((rows, heads), 7.0, device="cuda") if lse else None
    cache.handle(E).attention(ptr(q), heads, rows, ptr(ln), ptr(out), seq_ptr=ptr(sq), scale=scale, lse_ptr=ptr(ls),
                              weights_ptr=ptr(weights), stream=stream)
    torch.cuda.synchronize()
    return out, ls


def check_attention(cache, q, seq, lens, out, lse, scale=None, weights=None, before=None):
    scale = 1 / math.sqrt(cache.D) if scale is None else scale
    want, wlse, w, eo, ew = attention64(cache, q, seq, lens, scale)
    num = den = 0.0
    for i in range(len(lens)):
        err = (out[i].double() - want[i]).abs()
        assert bool((err <= eo[i]).all()), (i, seq[i], lens[i], float((err / eo[i].clamp(min=1e-30)).max()))
        num, den = num + float(err.square().sum()), den + float(want[i].square().sum())
        if lse is not None:
            assert torch.allclose(lse[i].double(), wlse[i], rtol=2e-6, atol=2e-5), (i, lens[i])
    # independent roundings: sqrt(D) of them a score of size ~1..8, 2^-24 each
    assert math.sqrt(num) <= 3e-6 * max(1e-30, math.sqrt(den)), math.sqrt(num / max(den, 1e-30))
    if weights is not None:
        # eight heads' weights at a time are added to the slot's: half a step, 2^-24, each time
        adds = 1 + -(-q.shape[1] // cache.kvheads // 8)
        total, bound = before.double(), torch.zeros_like(before, dtype=torch.float64)
        for i, (s, n) in enumerate(zip(seq, lens)):
            total[s, :, :n] += w[i]
            bound[s, :, :n] += ew[i] + adds * 2.0 ** -24 * (total[s, :, :n] + ew[i])
        err = (weights.double() - total).abs()
        assert bool((err <= bound).all()), float((err - bound).max())


SHAPES = [  # kind, heads, kvheads, D, page, lens
    ("f16", 32, 4, 128, 16, [1, 15, 16, 17, 31, 32, 33, 255, 0, 640]),
    ("bf16", 32, 4, 128, 16, [0, 1, 2, 63, 64, 65, 127, 129, 1023, 4096]),
    ("f32", 32, 4, 128, 16, [0, 1, 8, 9, 64, 500, 1025]),
    ("bf16", 4, 2, 64, 7, [13, 0, 100, 301]),
    ("f16", 6, 2, 96, 24, [5, 48, 777]),
    ("f32", 12, 4, 96, 24, [0, 3, 50, 333]),
    ("bf16", 32, 1, 80, 1, [1, 40, 130]),
    ("f16", 32, 1, 256, 250, [249, 250, 251, 600]),
    ("f32", 9, 3, 256, 5, [0, 31, 97]),
    ("f32", 16, 1, 4, 3, [1, 10, 70]),
    ("f16", 2, 2, 8, 16, [1, 33]),
    ("bf16", 64, 2, 192, 64, [129, 700]),
    ("bf16", 17, 1, 72, 16, [18, 260]),
    ("f16", 5, 5, 32, 128, [1, 1000]),
    ("bf16", 8, 1, 128, 64, [20000]),
    ("f16", 8, 1, 128, 64, [70001]),
    ("f32", 8, 1, 64, 64, [30011]),
]


@pytest.mark.parametrize("kind,heads,kvheads,D,page,lens", SHAPES)
def test_attention_matches_the_formula(cuda_engine, torch_cuda, kind, heads, kvheads, D, page, lens):
    cache = Cache(kind, kvheads, D, page, lens, seed=D + page)
    g = torch.Generator().manual_seed(5)
    q = (torch.randn(len(lens), heads, D, generator=g) * (0.5 + 2 * torch.rand(1, heads, 1, generator=g))).cuda()
    out, lse = run_attention(cuda_engine, cache, q, None, lens)
    check_attention(cache, q, range(len(lens)), lens, out, lse)
    again, _ = run_attention(cuda_engine, cache, q, None, lens, lse=False)
    assert torch.equal(out, again)  # the same bits
    weights = torch.rand(len(lens), kvheads, cache.cap, generator=g).cuda()
    before = weights.clone()
    out, lse = run_attention(cuda_engine, cache, q, None, lens, weights=weights)
    check_attention(cache, q, range(len(lens)), lens, out, lse, weights=weights, before=before)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f32", 64), ("f16", 96)])
def test_rows_of_one_sequence_and_padding(cuda_engine, torch_cuda, kind, D):
    """A prompt's last tokens beside decode tokens, in any order; rows of sequences that do not exist are
    left as they were."""
    cache = Cache(kind, 2, D, 16, [700, 64, 0, 33], seed=3)
    seq = [0, 1, 0, -1, 0, 3, 1, 9, 2]
    lens = [698, 64, 699, 5, 700, 33, 60, 12, 0]
    q = torch.randn(len(seq), 12, D, generator=torch.Generator().manual_seed(1)).cuda()
    real = [i for i, s in enumerate(seq) if 0 <= s < 4]
    for with_weights in (False, True):
        weights = torch.rand(4, 2, cache.cap, generator=torch.Generator().manual_seed(2)).cuda() if with_weights else None
        before = weights.clone() if with_weights else None
        out, lse = run_attention(cuda_engine, cache, q, seq, lens, weights=weights)
        check_attention(cache, q[real], [seq[i] for i in real], [lens[i] for i in real], out[real], lse[real],
                        weights=weights, before=before)
        for i in (3, 7):
            assert bool((out[i] == 7).all()) and bool((lse[i] == 7).all())
        if with_weights:
            w1 = before.clone()
            out2, _ = run_attention(cuda_engine, cache, q, seq, lens, weights=w1)
            assert torch.equal(w1, weights) and torch.equal(out, out2)  # rows of one sequence add in call order


def test_scale_and_extreme_scores(cuda_engine, torch_cuda):
    cache = Cache("bf16", 2, 64, 16, [50, 200], seed=9)
    q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(1)).cuda()
    for scale in (0.25, -0.5, 4.0):
        out, lse = run_attention(cuda_engine, cache, q, None, [50, 200], scale=scale)
        check_attention(cache, q, range(2), [50, 200], out, lse, scale=scale)
    # a slot masked by the type's lowest value has no weight, and alone leaves nothing
    t = cache.table[0].long()
    lowest = torch.finfo(torch.bfloat16).min
    at = torch.arange(50, device="cuda")
    cache.k[t[at[:7] // 16], :, at[:7] % 16] = lowest
    ones = torch.full_like(q, 4.0)
    weights = torch.zeros(2, 2, cache.cap, device="cuda")
    out, lse = run_attention(cuda_engine, cache, ones, None, [50, 200], weights=weights)
    assert bool(torch.isfinite(out).all()) and bool((weights[0, :, :7] == 0).all())
    k = cache.rows(0, 50).double()[7:, 0]
    p = torch.softmax((k.sum(1) * 4) / 8, 0)
    want = p @ cache.rows(0, 50, "v").double()[7:, 0]
    assert torch.allclose(out[0, 0].double(), want, rtol=1e-4, atol=1e-4)
    out, lse = run_attention(cuda_engine, cache, ones, None, [7, 1], weights=weights)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -float("inf")).all())
    assert bool((weights[0, :, :7] == 0).all())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_bad_pages_and_lengths_stay_in_bounds(cuda_engine, torch_cuda, kind):
    cache = Cache(kind, 2, 64, 16, [100, 90, 40, 200], seed=4)
    q = torch.randn(4, 8, 64, generator=torch.Generator().manual_seed(1)).cuda()
    weights = torch.rand(4, 2, cache.cap, generator=torch.Generator().manual_seed(2)).cuda()
    before = weights.clone()
    good = cache.table.clone()
    cache.table[1, 3] = cache.n_pages      # within the 90 slots
    cache.table[2, 5] = 1 << 30            # behind the 40 slots: never looked at
    lens = [100, 90, 40, cache.cap + 1]
    out, lse = run_attention(cuda_engine, cache, q, None, lens, weights=weights)
    for i in (1, 3):
        assert bool(out[i].isnan().all()) and bool(lse[i].isnan().all())
        assert torch.equal(weights[i], before[i])
    check_attention(cache, q[[0, 2]], [0, 2], [100, 40], out[[0, 2]], lse[[0, 2]])
    # append skips what has no slot
    k, v = (torch.randn(5, 2, 64, device="cuda") for _ in range(2))
    seq = torch.tensor([0, 1, 3, 7, -1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([100, 50, cache.cap, 3, 3], dtype=torch.int32, device="cuda")
    k0, v0 = cache.k.clone(), cache.v.clone()
    cache.handle(cuda_engine).append(ptr(k), ptr(v), 5, ptr(pos), seq_ptr=ptr(seq), weights_ptr=ptr(weights))
    torch.cuda.synchronize()
    at = (int(good[0, 100 // 16]), slice(None), 100 % 16)
    assert torch.equal(cache.k[at], k[0].to(DTYPE[kind])) and torch.equal(cache.v[at], v[0].to(DTYPE[kind]))
    cache.k[at], cache.v[at] = k0[at], v0[at]
    assert torch.equal(cache.k.nan_to_num(9), k0.nan_to_num(9)) and torch.equal(cache.v.nan_to_num(9), v0.nan_to_num(9))
    # eviction leaves a bad sequence alone
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept = torch.zeros(4, 2, 30, dtype=torch.int32, device="cuda")
    new = torch.zeros(4, dtype=torch.int32, device="cuda")
    weights = before.clone()
    bad = cache.rows(0, 100).clone()
    dst = good.clone()
    dst[0, 1] = cache.n_pages  # a bad page among those it would write
    cache.handle(cuda_engine).evict(ptr(weights), ptr(ln), 30, 4, ptr(kept), ptr(new), dst_table_ptr=ptr(dst))
    torch.cuda.synchronize()
    assert new.tolist() == [100, 90, 30, cache.cap + 1]
    assert bool((kept[[0, 1, 3]] == -1).all())
    assert torch.equal(weights[[0, 1, 3]], before[[0, 1, 3]]) and torch.equal(cache.rows(0, 100), bad)
    assert kept[2, 0].tolist() == evict64(before[2, 0], 40, 30, 4)


def test_offsets_beyond_32_bits(cuda_engine, torch_cuda):
    """Pools of more than 2^32 values; the sequence's pages lie at the far end."""
    KH, page, D, n_pages = 4, 64, 128, 132000  # 4.3e9 values
    k = torch.empty(n_pages, KH, page, D, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    tail = Cache("f16", KH, D, page, [300, 1000], spare=0, seed=8)
    base = n_pages - tail.n_pages
    k[base:], v[base:] = tail.k, tail.v
    near = tail.table.clone()
    tail.table += base
    tail.k, tail.v, tail.n_pages = k, v, n_pages
    assert int(tail.table.max()) * KH * page * D > 2 ** 32
    q = torch.randn(2, 32, D, generator=torch.Generator().manual_seed(1)).cuda()
    weights = torch.rand(2, KH, tail.cap, generator=torch.Generator().manual_seed(2)).cuda()
    before = weights.clone()
    out, lse = run_attention(cuda_engine, tail, q, None, [300, 1000], weights=weights)
    check_attention(tail, q, range(2), [300, 1000], out, lse, weights=weights, before=before)
    row = torch.randn(2, 1, KH, D, device="cuda")
    pos = torch.tensor([300], dtype=torch.int32, device="cuda")
    tail.handle(cuda_engine).append(ptr(row[0]), ptr(row[1]), 1, ptr(pos))
    torch.cuda.synchronize()
    assert torch.equal(tail.rows(0, 301)[300], row[0, 0].half()) and torch.equal(tail.rows(0, 301, "v")[300], row[1, 0].half())
    # evict from the far end to pages at the start of the pool
    kept = torch.zeros(2, KH, 200, dtype=torch.int32, device="cuda")
    ln = torch.tensor([301, 1000], dtype=torch.int32, device="cuda")
    old = [tail.rows(s, int(n)).clone() for s, n in enumerate(ln)]
    dst = near % 64
    dst[0], dst[1] = torch.arange(tail.max_pages), torch.arange(tail.max_pages) + tail.max_pages
    wout = torch.zeros_like(weights)
    tail.handle(cuda_engine).evict(ptr(weights), ptr(ln), 200, 20, ptr(kept), ptr(ln), weights_out_ptr=ptr(wout),
                                   dst_table_ptr=ptr(dst))
    torch.cuda.synchronize()
    assert ln.tolist() == [200, 200]
    for s, n in enumerate((301, 1000)):
        for h in range(KH):
            want = evict64(weights[s, h], n, 200, 20)
            assert kept[s, h].tolist() == want
            assert torch.equal(tail.rows(s, 200, table=dst)[:, h], old[s][want, h])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kvheads,D,page,rows", [(4, 128, 16, 1), (2, 64, 5, 37), (1, 8, 1, 3), (3, 80, 24, 700), (2, 256, 64, 65)])
def test_append_rounds_to_nearest(cuda_engine, torch_cuda, kind, kvheads, D, page, rows):
    cache = Cache(kind, kvheads, D, page, [4, 0, 9], cap=rows + 9, seed=1)
    g = torch.Generator().manual_seed(rows)
    k, v = (torch.randn(3 * rows, kvheads, D, generator=g).cuda() * 3 for _ in range(2))
    seq = torch.arange(3).repeat_interleave(rows)
    pos = torch.tensor(cache.lens)[seq] + torch.arange(rows).repeat(3)
    mix = torch.randperm(3 * rows, generator=g)
    seq, pos = seq[mix].to(torch.int32).cuda(), pos[mix].to(torch.int32).cuda()
    weights = torch.rand(3, kvheads, cache.cap, generator=g).cuda()
    wk, wv, ww = cache.k.clone(), cache.v.clone(), weights.clone()
    at = cache.table[seq.long(), (pos // page).long()].long()
    wk[at, :, (pos % page).long()] = k.to(DTYPE[kind])
    wv[at, :, (pos % page).long()] = v.to(DTYPE[kind])
    ww[seq.long(), :, pos.long()] = 0
    cache.handle(cuda_engine).append(ptr(k), ptr(v), 3 * rows, ptr(pos), seq_ptr=ptr(seq), weights_ptr=ptr(weights))
    torch.cuda.synchronize()
    bits = {4: torch.int32, 2: torch.int16}[wk.element_size()]
    assert torch.equal(cache.k.view(bits), wk.view(bits)) and torch.equal(cache.v.view(bits), wv.view(bits))
    assert torch.equal(weights, ww)


EVICT = [  # kind, kvheads, D, page, lens, keep, recent
    ("f16", 4, 128, 16, [100, 64, 63, 65, 0, 1, 400], 64, 8),
    ("bf16", 2, 64, 7, [50, 51, 500], 50, 50),
    ("f32", 1, 96, 24, [1000, 33], 33, 0),
    ("f16", 3, 80, 1, [10, 200], 1, 0),
    ("bf16", 1, 256, 250, [3001, 2000], 1999, 17),
    ("f32", 2, 4, 3, [90, 4], 5, 1),
    ("f16", 1, 128, 64, [20011], 4999, 128),
    ("bf16", 2, 128, 32, [70000, 100], 30000, 1),
    ("f32", 2, 256, 16, [1100], 1024, 1024),
]


@pytest.mark.parametrize("how", ["in place", "elsewhere"])
@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
@pytest.mark.parametrize("kind,kvheads,D,page,lens,keep,recent", EVICT)
def test_evict_keeps_the_largest_weights(cuda_engine, torch_cuda, kind, kvheads, D, page, lens, keep, recent, values, how):
    S = len(lens)
    cache = Cache(kind, kvheads, D, page, lens, seed=keep, spare=S * (-(-max(keep, max(lens)) // page)))
    g = torch.Generator().manual_seed(keep + recent)
    w = torch.exp(3 * torch.randn(S, kvheads, cache.cap, generator=g))
    if values == "ties":
        w = torch.floor(torch.rand(S, kvheads, cache.cap, generator=g) * 3) * 0.5 * (1 - 2 * (w > 30).float())
    elif values == "odd":
        odd = torch.tensor([0.0, -0.0, float("nan"), float("inf"), -float("inf"), -1.5, 1e-42, 3e38])
        pick = torch.randint(0, 16, w.shape, generator=g)
        w = torch.where(pick < 8, odd[pick % 8], w)
    weights = w.cuda()
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept = torch.zeros(S, kvheads, keep, dtype=torch.int32, device="cuda")
    old = {p: [cache.rows(s, n, p).clone() for s, n in enumerate(lens)] for p in "kv"}
    free = sorted(set(range(cache.n_pages)) - set(cache.table.flatten().tolist()))
    if how == "in place":
        dst, wout, new = cache.table, weights, lens_d
        cache.handle(cuda_engine).evict(ptr(weights), ptr(lens_d), keep, recent, ptr(kept), ptr(lens_d))
    else:
        dst = torch.tensor(free[: S * cache.max_pages], dtype=torch.int32).reshape(S, cache.max_pages).cuda()
        wout, new = torch.full_like(weights, 5.0), torch.zeros_like(lens_d)
        cache.handle(cuda_engine).evict(ptr(weights), ptr(lens_d), keep, recent, ptr(kept), ptr(new),
                                        weights_out_ptr=ptr(wout), dst_table_ptr=ptr(dst))
    torch.cuda.synchronize()
    assert new.tolist() == [min(n, keep) for n in lens]
    bits = {4: torch.int32, 2: torch.int16}[cache.k.element_size()]
    for s, n in enumerate(lens):
        m = min(n, keep)
        for h in range(kvheads):
            want = evict64(w[s, h], n, keep, recent)
            assert kept[s, h].tolist() == want + [-1] * (keep - m), (s, h)
            assert torch.equal(wout[s, h, :m].view(torch.int32), w[s, h][want].cuda().view(torch.int32))
            if how == "elsewhere":
                assert bool((wout[s, h, m:] == 5).all())
            for p in "kv":
                assert torch.equal(cache.rows(s, m, p, table=dst)[:, h].view(bits), old[p][s][want, h].view(bits)), (s, h, p)
        if how == "elsewhere":
            for p in "kv":
                assert torch.equal(cache.rows(s, n, p).view(bits), old[p][s].view(bits))


def test_decoding_with_a_bounded_cache(cuda_engine, torch_cuda):
    """append, attention with weights and eviction in turn, as a serving loop calls them: two sequences
    of their own lengths past a budget of 40 slots, against the same loop in 64 bits."""
    KH, D, heads, budget, recent = 2, 64, 8, 40, 6
    cache = Cache("f16", KH, D, 8, [0, 0], cap=64, seed=1)
    cache.k.zero_(), cache.v.zero_()
    h = cache.handle(cuda_engine)
    g = torch.Generator().manual_seed(4)
    weights = torch.zeros(2, KH, cache.cap, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    kept = torch.zeros(2, KH, budget, dtype=torch.int32, device="cuda")
    ref = [{"k": [[] for _ in range(KH)], "v": [[] for _ in range(KH)], "w": [[] for _ in range(KH)]} for _ in range(2)]
    evictions = 0
    for step in range(90):
        live = [0, 1] if step % 3 else [1]
        seq = torch.tensor(live, dtype=torch.int32, device="cuda")
        k, v = (torch.randn(len(live), KH, D, generator=g).cuda() for _ in range(2))
        q = torch.randn(len(live), heads, D, generator=g).cuda() * 2
        pos = lens[seq.long()].contiguous()
        h.append(ptr(k), ptr(v), len(live), ptr(pos), seq_ptr=ptr(seq), weights_ptr=ptr(weights))
        lens[seq.long()] += 1
        row_lens = lens[seq.long()].contiguous()
        out, lse = torch.zeros(len(live), heads, D, device="cuda"), torch.zeros(len(live), heads, device="cuda")
        h.attention(ptr(q), heads, len(live), ptr(row_lens), ptr(out), seq_ptr=ptr(seq), lse_ptr=ptr(lse),
                    weights_ptr=ptr(weights))
        for i, s in enumerate(live):
            for kh in range(KH):
                ref[s]["k"][kh].append(k[i, kh].half().double())
                ref[s]["v"][kh].append(v[i, kh].half().double())
                ref[s]["w"][kh].append(0.0)
                K, V = torch.stack(ref[s]["k"][kh]), torch.stack(ref[s]["v"][kh])
                p = torch.softmax(q[i, kh * 4:kh * 4 + 4].double() @ K.T / 8, 1)
                err = (out[i, kh * 4:kh * 4 + 4].double() - p @ V).abs().max()
                assert float(err) < 2e-5, (step, s, kh)  # f32 scores of size up to ~16
                ref[s]["w"][kh] = [a + b for a, b in zip(ref[s]["w"][kh], p.sum(0).tolist())]
                got = weights[s, kh, : len(ref[s]["w"][kh])].double().cpu()
                assert torch.allclose(got, torch.tensor(ref[s]["w"][kh], dtype=torch.float64), rtol=2e-5, atol=1e-6)
        if int(lens.max()) >= 56:
            before = lens.clone()
            snapshot = weights.clone()
            h.evict(ptr(weights), ptr(lens), budget, recent, ptr(kept), ptr(lens))
            torch.cuda.synchronize()
            evictions += 1
            for s in range(2):
                n = int(before[s])
                assert int(lens[s]) == min(n, budget)
                for kh in range(KH):
                    want = evict64(snapshot[s, kh], n, budget, recent)
                    assert kept[s, kh, : len(want)].tolist() == want
                    for f in "kvw":
                        ref[s][f][kh] = [ref[s][f][kh][j] for j in want]
    assert evictions >= 2


def test_captured_calls_replay_on_new_data(cuda_engine, torch_cuda):
    """append, attention and eviction in one graph, replayed with other lengths and rows; two graphs of
    different caches at once on two streams."""
    def make(seed):
        cache = Cache("bf16", 2, 128, 16, [200, 90, 0], cap=512, seed=seed)
        d = {"cache": cache, "lens": torch.tensor([200, 90, 0], dtype=torch.int32, device="cuda"),
             "k": torch.randn(3, 2, 128, device="cuda"), "v": torch.randn(3, 2, 128, device="cuda"),
             "q": torch.randn(3, 16, 128, device="cuda"), "out": torch.zeros(3, 16, 128, device="cuda"),
             "lse": torch.zeros(3, 16, device="cuda"), "w": torch.rand(3, 2, cache.cap, device="cuda"), "kept": torch.zeros(3, 2, 100, dtype=torch.int32, device="cuda"),
             "new": torch.zeros(3, dtype=torch.int32, device="cuda")}
        d["after"] = d["lens"] + 1
        return d

    def step(d, stream):
        h = d["cache"].handle(cuda_engine)
        h.append(ptr(d["k"]), ptr(d["v"]), 3, ptr(d["lens"]), weights_ptr=ptr(d["w"]), stream=stream)
        h.attention(ptr(d["q"]), 16, 3, ptr(d["after"]), ptr(d["out"]), lse_ptr=ptr(d["lse"]), weights_ptr=ptr(d["w"]),
                    stream=stream)
        h.evict(ptr(d["w"]), ptr(d["after"]), 100, 10, ptr(d["kept"]), ptr(d["new"]), stream=stream)

    names = ("out", "lse", "w", "kept", "new")
    graphs = []
    for seed in (1, 2):
        d, same = make(seed), make(seed)
        for name in ("k", "v", "q", "w"):
            same[name].copy_(d[name])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step(d, torch.cuda.current_stream().cuda_stream)
        graphs.append((g, d, same, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for round_ in range(3):
        for _, d, same, _ in graphs:
            for x in (d, same):
                x["lens"].copy_(torch.tensor([120 + 7 * round_, 33, 5 * round_]))
                x["after"].copy_(x["lens"] + 1)
        torch.cuda.synchronize()
        for g, _, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for _, d, same, _ in graphs:
            step(same, None)
            torch.cuda.synchronize()
            for name in names:
                assert torch.equal(d[name].nan_to_num(3), same[name].nan_to_num(3)), (round_, name)
            for pool in "kv":
                assert torch.equal(getattr(d["cache"], pool).nan_to_num(3), getattr(same["cache"], pool).nan_to_num(3))


def test_no_rows_and_host_pointers(cuda_engine, torch_cuda):
    cache = Cache("f16", 2, 64, 16, [10], seed=1)
    h = cache.handle(cuda_engine)
    h.attention(None, 4, 0, None, None)
    h.append(None, None, 0, None)
    q, out = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 4, 64, device="cuda")
    ln = torch.tensor([3], dtype=torch.int32)  # host memory
    with pytest.raises(cuda_engine.QwenCudaError, match="len is not device memory"):
        h.attention(ptr(q), 4, 1, ptr(ln), ptr(out))
    assert bool((out == 0).all())


@pytest.mark.parametrize("kind,heads,kvheads,D,page,rows,hi,pad", [
    ("bf16", 32, 4, 128, 16, 64, 900, 0),   # more blocks than fit at once: the longest rows first
    ("f16", 32, 4, 128, 16, 8, 9000, 0),    # clusters of other than a power of two
    ("f32", 6, 2, 64, 24, 130, 300, 5),     # more rows than are sorted
    ("bf16", 10, 1, 32, 3, 700, 70, 1),
    ("f16", 24, 8, 256, 128, 40, 700, 2),
])
def test_many_rows(cuda_engine, torch_cuda, kind, heads, kvheads, D, page, rows, hi, pad):
    """Lengths all over the range, empty ones among them, padding behind; with and without weights."""
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, hi + 1, (rows,), generator=g).tolist()
    lens[0], lens[-1], lens[rows // 2] = hi, 0, 1
    cache = Cache(kind, kvheads, D, page, lens, seed=2)
    q = torch.randn(rows + pad, heads, D, generator=g).cuda()
    seq = torch.randperm(rows, generator=g).tolist()
    real = [lens[s] for s in seq]
    weights = torch.rand(rows, kvheads, cache.cap, generator=g).cuda()
    before = weights.clone()
    out, lse = run_attention(cuda_engine, cache, q, seq + [-1] * pad, real + [0] * pad, weights=weights)
    check_attention(cache, q[:rows], seq, real, out[:rows], lse[:rows], weights=weights, before=before)
    assert bool((out[rows:] == 7).all()) and bool((lse[rows:] == 7).all())
    again, _ = run_attention(cuda_engine, cache, q, seq + [-1] * pad, real + [0] * pad)
    assert torch.equal(again, out)


def test_many_rows_of_one_sequence_give_their_weights_in_any_call(cuda_engine, torch_cuda):
    """A prompt's 150 tokens in one call, and each in a call of its own: the same outputs, and weights that
    differ by the additions' roundings only (one a call: 150 half steps)."""
    cache = Cache("f16", 2, 64, 16, [400, 30], seed=5)
    q = torch.randn(150, 8, 64, generator=torch.Generator().manual_seed(1)).cuda()
    seq, lens = [0] * 150, list(range(251, 401))
    one, many = (torch.zeros(2, 2, cache.cap, device="cuda") for _ in range(2))
    out, _ = run_attention(cuda_engine, cache, q, seq, lens, weights=one)
    for i in range(150):
        row, _ = run_attention(cuda_engine, cache, q[i:i + 1].contiguous(), [0], [lens[i]], weights=many)
        assert torch.allclose(row[0], out[i], rtol=0, atol=2e-6)
    assert bool(((one - many).abs() <= 1e-5 * many.abs() + 1e-9).all())
    assert bool((one[1] == 0).all())


def test_a_slot_named_twice_holds_one_of_the_rows(cuda_engine, torch_cuda):
    """Rows of a call have different slots; where they do not, every value is one of theirs."""
    cache = Cache("bf16", 2, 64, 16, [5], cap=32, seed=1)
    k, v = torch.ones(4, 2, 64, device="cuda"), torch.ones(4, 2, 64, device="cuda")
    k *= torch.arange(1, 5, device="cuda")[:, None, None]
    seq, pos = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.full((4,), 7, dtype=torch.int32, device="cuda")
    cache.handle(cuda_engine).append(ptr(k), ptr(v), 4, ptr(pos), seq_ptr=ptr(seq))
    torch.cuda.synchronize()
    got = cache.rows(0, 8)[7].float()
    assert bool(((got >= 1) & (got <= 4) & (got == got.round())).all())


@pytest.mark.parametrize("S,n,keep,recent", [(150, 41500, 30001, 77), (1, 400003, 123457, 1000)])
def test_evict_of_more_slots_than_are_held(cuda_engine, torch_cuda, S, n, keep, recent):
    """Sequences whose weights do not fit the selection's shared memory, alone and with many short ones."""
    lens = [n] + [100] * (S - 1)
    cache = Cache("f32", 1, 4, 64, lens, seed=6)
    w = torch.floor(torch.rand(S, 1, cache.cap, generator=torch.Generator().manual_seed(1)) * 50000)  # ties
    weights, lens_d = w.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept = torch.zeros(S, 1, keep, dtype=torch.int32, device="cuda")
    old = cache.rows(0, n, "v").clone()
    cache.handle(cuda_engine).evict(ptr(weights), ptr(lens_d), keep, recent, ptr(kept), ptr(lens_d))
    torch.cuda.synchronize()
    want = torch.tensor(evict64(w[0, 0], n, keep, recent))
    assert lens_d.tolist() == [keep] + [100] * (S - 1)
    assert torch.equal(kept[0, 0].long().cpu(), want)
    assert torch.equal(weights[0, 0, :keep].cpu(), w[0, 0][want])
    assert torch.equal(cache.rows(0, keep, "v")[:, 0], old[want.cuda(), 0])


def test_calls_at_once_on_two_streams(cuda_engine, torch_cuda):
    """Calls on different caches from two streams, many times over, give what they give alone."""
    caches = [Cache(kind, 4, 128, 16, [300 + 50 * i for i in range(12)], seed=i) for i, kind in enumerate(("bf16", "f16"))]
    g = torch.Generator().manual_seed(1)
    qs = [torch.randn(12, 32, 128, generator=g).cuda() for _ in caches]
    alone = [run_attention(cuda_engine, c, q, None, c.lens)[0] for c, q in zip(caches, qs)]
    streams = [torch.cuda.Stream() for _ in caches]
    outs = [torch.zeros_like(a) for a in alone]
    lens = [torch.tensor(c.lens, dtype=torch.int32, device="cuda") for c in caches]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, q, o, ln, st in zip(caches, qs, outs, lens, streams):
            c.handle(cuda_engine).attention(ptr(q), 32, 12, ptr(ln), ptr(o), stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


@pytest.mark.parametrize("kind,heads,kvheads,D,page", [
    ("bf16", 32, 4, 128, 16),  # four rows share a sequence's tiles
    ("f16", 4, 4, 64, 16),     # one head a KV head: 32 rows
    ("f32", 6, 2, 96, 24),     # three: ten rows, 30 of 32 columns
    ("f16", 10, 2, 72, 7),     # five: six rows; pages of single lookups
    ("bf16", 34, 2, 32, 16),   # seventeen: one row, three parts of eight heads
    ("f32", 64, 2, 128, 64),
    ("bf16", 20, 1, 256, 16),  # twenty, two parts of eight at a time
    ("f16", 32, 1, 192, 3),
    ("f32", 2, 1, 256, 16),
    ("f32", 9, 3, 4, 5),
])
def test_rows_of_prompts_share_tiles(cuda_engine, torch_cuda, kind, heads, kvheads, D, page):
    """Many more rows than sequences: prompts' rows side by side, single rows between them, padding, rows of no
    positions, all in one call."""
    lens = [901, 64, 33, 0, 300]
    cache = Cache(kind, kvheads, D, page, lens, seed=6, cap=950)
    seq = [0] * 37 + [1] + [4] * 9 + [-1] * 2 + [2, 0, 2, 0] + [4] * 3 + [3] + [1] * 16 + [7] + [4] * 20
    want = [901 - 37 + 1 + i for i in range(37)] + [64] + list(range(1, 10)) + [5, 5] + [33, 900, 1, 0]
    want += [300, 0, 299] + [0] + list(range(49, 65)) + [3] + list(range(281, 301))
    q = torch.randn(len(seq), heads, D, generator=torch.Generator().manual_seed(1)).cuda()
    real = [i for i, s in enumerate(seq) if 0 <= s < 5]
    before = torch.rand(5, kvheads, cache.cap, generator=torch.Generator().manual_seed(2)).cuda()
    weights = before.clone()
    out, lse = run_attention(cuda_engine, cache, q, seq, want, weights=weights)
    check_attention(cache, q[real], [seq[i] for i in real], [want[i] for i in real], out[real], lse[real],
                    weights=weights, before=before)
    for i, s in enumerate(seq):
        if not 0 <= s < 5:
            assert bool((out[i] == 7).all()) and bool((lse[i] == 7).all())
    again, _ = run_attention(cuda_engine, cache, q, seq, want)
    assert torch.equal(again, out)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rows_that_share_tiles_do_not_share_what_is_wrong(cuda_engine, torch_cuda, kind):
    """Infinities, NaN and invalid pages behind a row's length, and a neighbour longer than the cache, leave
    the row as it is; rows that reach them are not finite."""
    cache = Cache(kind, 2, 64, 16, [200, 150], seed=8)
    q = torch.randn(32, 8, 64, generator=torch.Generator().manual_seed(1)).cuda()
    at = lambda s, j: (int(cache.table[s, j // 16]), slice(None), j % 16)
    cache.v[at(0, 190)] = float("inf")
    cache.v[at(0, 197)] = float("nan")
    cache.k[at(0, 198)] = float("nan")
    cache.table[1, 8] = cache.n_pages  # positions 128..143
    seq, over = [0] * 16 + [1] * 16, cache.cap + 1
    lens = [190, 191, 180, 200, 0, over, 190, 5, 199, 190, 100, 16, 0, 191, 198, 1]
    lens += [128, 129, 150, 127, 1, 17, 0, over, 128, 128, 64, 150, 144, 100, 16, 127]
    last = [190, 128]  # the longest that nothing is wrong with
    good = [i for i in range(32) if lens[i] <= last[seq[i]]]
    before = torch.rand(2, 2, cache.cap, generator=torch.Generator().manual_seed(2)).cuda()
    weights = before.clone()
    out, lse = run_attention(cuda_engine, cache, q, seq, lens, weights=weights)
    check_attention(cache, q[good], [seq[i] for i in good], [lens[i] for i in good], out[good], lse[good])
    for i in range(32):
        if i not in good:
            assert not bool(out[i].isfinite().any()), i
    for i in [i for i in range(32) if lens[i] == over or (seq[i] and lens[i] > 128)]:
        assert bool(out[i].isnan().all()) and bool(lse[i].isnan().all()), i
    # rows that reach an infinite value still have weights (their scores are finite); the others' are exact
    fine = [i for i in range(32) if i in good or (seq[i] == 0 and lens[i] <= 198)]
    w = before.double()
    _, _, ws, _, ew = attention64(cache, q[fine], [seq[i] for i in fine], [lens[i] for i in fine], 0.125)
    bound = torch.zeros_like(w)
    for i, x, e in zip(fine, ws, ew):
        w[seq[i], :, :lens[i]] += x
        bound[seq[i], :, :lens[i]] += e + 2.0 ** -23 * (w[seq[i], :, :lens[i]] + e)
    assert bool(((weights.double() - w).abs() <= bound).all())
