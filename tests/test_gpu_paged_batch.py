"""Batches with a paged cache (qc_batch_create_paged), eviction in them (qc_batch_evict) and the log
probabilities of their logits (qc_batch_logprobs, qc_engine_logprobs)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 30


@pytest.fixture(scope="module")
def model(cuda_engine, tools):
    img = tools.synth_gguf(tools.TINY)
    return img, cuda_engine.Engine(img, 256), tools.TINY


def prompts(spec, lens, seed=3):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, spec.vocab, n).tolist() for n in lens]


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("weights", [False, True])
def test_f32_pages_give_the_contiguous_caches_logits(cuda_engine, oracle, model, page, weights):
    """Prompts whole, interleaved and across the pass size, then decode steps, each row against the oracle on
    its sequence alone (the decode path's tolerance; 1e-3 as for contiguous caches)."""
    img, eng, spec = model
    lens = [5, 1, 150, 40]
    b = cuda_engine.Batch.paged(eng, 4, 256, F32, page, 4 * (-(-200 // page)), weights)
    refs = [oracle.Model(img, 256) for _ in range(4)]
    ps = prompts(spec, lens)

    def ref(q, toks):
        for t in toks:
            out = refs[q].forward(t)
        return out

    total = b.cache(0)[1]
    rows = b.forward([2] * 150 + [0] * 5, ps[2] + ps[0])
    got = [(2, rows[0]), (0, rows[1])]
    order = [(1, ps[1][0])] + [(3, t) for t in ps[3][:20]]
    rows = b.forward([q for q, _ in order] + [3] * 20, [t for _, t in order] + ps[3][20:])
    got += [(1, rows[0]), (3, rows[1])]
    for q, row in got:
        want = ref(q, ps[q])
        assert np.abs(row - want).max() < 1e-3 and int(np.argmax(row)) == int(np.argmax(want)), q
    rng = np.random.default_rng(1)
    for step in range(6):
        perm, toks = rng.permutation(4).tolist(), rng.integers(0, spec.vocab, 4).tolist()
        for row, q, t in zip(b.forward(perm, toks), perm, toks):
            assert np.abs(row - refs[q].forward(t)).max() < 1e-3, (step, q)
    assert [b.cache(q)[0] for q in range(4)] == [n + 6 for n in lens] == [b.position(q) for q in range(4)]
    used = sum(-(-(n + 6) // page) for n in lens)
    assert b.cache(0)[1] == total - used
    b.reset(2)
    assert b.cache(2)[0] == 0 and b.cache(0)[1] == total - used + -(-156 // page)
    refs[2].reset()
    want = ref(2, ps[3])
    assert np.abs(b.forward([2] * 40, ps[3])[0] - want).max() < 1e-3
    if weights:  # a budget nobody exceeds changes nothing
        before = [b.cache(q) for q in range(4)]
        b.evict(200, 10)
        assert [b.cache(q) for q in range(4)] == before
    b.close()


@pytest.mark.parametrize("kind", [F16, BF16])
def test_16_bit_pages_stay_near(cuda_engine, model, kind):
    """Keys and values rounded once: relative 2^-11 (f16) or 2^-8 (bf16) of each, so the logits may move by
    about that times their own size; held to eight times it (two layers, keys and values, top of sums)."""
    _, eng, spec = model
    ps = prompts(spec, [60, 33])
    a = cuda_engine.Batch(eng, 2, 256)
    b = cuda_engine.Batch.paged(eng, 2, 256, kind, 16, 32)
    seqs, toks = [0] * 60 + [1] * 33, ps[0] + ps[1]
    want, got = a.forward(seqs, toks), b.forward(seqs, toks)
    assert np.abs(got - want).max() < 8 * (2.0 ** -11 if kind == F16 else 2.0 ** -8) * np.abs(want).max()
    assert not np.array_equal(got, want)
    assert b.stats()["kv_bytes"] == 2 * spec.layers * 32 * 16 * spec.kvheads * spec.head_dim * 2
    # the chat loop on the device takes pages as it goes, and equals a loop driven from the host
    mk = lambda: [cuda_engine.Sampler(7 + i, 0.8, 20, 0.9) for i in range(2)]
    ids = b.decode_sample(mk(), [0, 1], 20)
    assert b.cache(0)[0] == 80 and b.cache(1)[0] == 53
    c = cuda_engine.Batch.paged(eng, 2, 256, kind, 16, 32)
    c.forward(seqs, toks)
    smp = mk()
    for step in range(20):
        one = c.sample(smp, [0, 1])
        assert one.tolist() == ids[step].tolist()
        c.forward([0, 1], one)


def test_eviction_bounds_the_cache(cuda_engine, model):
    """A prompt fed whole and token by token keeps the same slots (the weights are the same up to rounding),
    whatever the page size; what stays is what the sequence goes on with."""
    _, eng, spec = model
    prompt = prompts(spec, [120], 9)[0]
    runs = []
    for page, whole in ((16, True), (16, False), (7, True)):
        b = cuda_engine.Batch.paged(eng, 2, 256, F32, page, 80, weights=True)
        free0 = b.cache(0)[1]
        if whole:
            b.forward([1] * 120, prompt)
        else:
            for t in prompt:
                b.forward([1], [t])
        b.forward([0] * 10, prompt[:10])
        b.evict(48, 12)
        assert b.cache(1)[0] == 48 and b.position(1) == 120 and b.cache(0)[0] == 10
        assert b.cache(0)[1] == free0 - -(-48 // page) - -(-10 // page)
        rows = [b.forward([1, 0], [t, t])for t in prompt[:8]]
        assert b.cache(1)[0] == 56 and b.position(1) == 128
        b.evict(50, 50, seq=1)  # the last 50 only
        assert b.cache(1)[0] == 50 and b.cache(0)[0] == 18
        rows.append(b.forward([1, 0], [5, 5]))
        runs.append(np.stack(rows))
        b.close()
    scale = np.abs(runs[0]).max()
    for other in runs[1:]:
        assert np.abs(other - runs[0]).max() < 1e-3 * scale
    full = cuda_engine.Batch(eng, 2, 256)
    full.forward([1] * 120, prompt)
    full.forward([0] * 10, prompt[:10])
    rows = [full.forward([1, 0], [t, t]) for t in prompt[:8]]
    assert np.abs(runs[0][7][0] - rows[7][0]).max() > 1e-3 * scale  # the evicted sequence has forgotten something
    for i in range(8):
        assert np.abs(runs[0][i][1] - rows[i][1]).max() < 1e-3  # the other one nothing


def test_a_full_cache_refuses_and_changes_nothing(cuda_engine, model):
    _, eng, spec = model
    b = cuda_engine.Batch.paged(eng, 3, 256, F16, 16, 6, weights=True)
    ps = prompts(spec, [40, 40])
    first = b.forward([0] * 40, ps[0])  # 3 pages
    with pytest.raises(cuda_engine.QwenCudaError, match="3 free pages, 4 are needed") as ei:
        b.forward([1] * 49, ps[1] + ps[0][:9])
    assert ei.value.code == cuda_engine.ERR_CONTEXT
    with pytest.raises(cuda_engine.QwenCudaError, match="free pages"):
        b.decode_sample([cuda_engine.Sampler(1, 0.0, 0, 1.0)], [0], 100)
    assert b.cache(1) == (0, 3) and b.cache(0) == (40, 3) and b.position(0) == 40
    b.forward([1] * 40, ps[1])
    with pytest.raises(cuda_engine.QwenCudaError, match="0 free pages"):
        b.forward([0] * 9, ps[1][:9])
    b.evict(16, 8, seq=0)  # two pages come back
    assert b.cache(0) == (16, 2)
    b.forward([0] * 9, ps[1][:9])
    assert b.cache(0) == (25, 1)
    b.reset()
    assert b.cache(0) == (0, 6)
    again = b.forward([2] * 40, ps[0])
    assert np.abs(again - first).max() < 1e-4
    for bad, match in ((dict(keep=0, recent=0), "at least 1"), (dict(keep=4, recent=5), "at most keep"),
                       (dict(keep=4, recent=1, seq=3), "sequence index")):
        with pytest.raises(cuda_engine.QwenCudaError, match=match):
            b.evict(**bad)
    plain = cuda_engine.Batch(eng, 1, 64)
    for call in (lambda: plain.evict(4, 1), lambda: plain.cache(0),
                 lambda: cuda_engine.Batch.paged(eng, 1, 64, F16, 16, 8).evict(4, 1)):
        with pytest.raises(cuda_engine.QwenCudaError, match="paged batch"):
            call()
    for bad in ((1, 64, 12, 16, 8), (1, 64, F16, 0, 8), (1, 64, F16, 16, 0), (0, 64, F16, 16, 8), (1, 300, F16, 16, 8)):
        with pytest.raises(cuda_engine.QwenCudaError):
            cuda_engine.Batch.paged(eng, *bad)


def check_logprobs(logits, ids, top, got):
    lp, ent, ti, tl = got
    x = logits.astype(np.float64)
    want = x - (np.log(np.exp(x - x.max()).sum()) + x.max())
    assert np.abs(lp - want[list(ids)]).max(initial=0) < 1e-5 and abs(ent + (np.exp(want) * want).sum()) < 1e-5
    order = np.lexsort((np.arange(x.size), -x))[:top]
    assert ti.tolist() == order.tolist() and np.abs(tl - want[order]).max(initial=0) < 1e-5


def test_logprobs_of_an_engine_and_a_batch(cuda_engine, model):
    """f32 log probabilities of logits of size up to ~10: 2^-23 of that and of the sum's logarithm."""
    img, eng, spec = model
    own = cuda_engine.Engine(img, 64)
    with pytest.raises(cuda_engine.QwenCudaError, match="previous forward"):
        own.logprobs([1])
    logits = own.forward_tokens([3, 9, 4])
    check_logprobs(logits, [7, 0, 511], 20, own.logprobs([7, 0, 511], 20))
    check_logprobs(logits, [], 0, own.logprobs())
    assert np.array_equal(own.forward(5), cuda_engine.Engine(img, 64).forward_tokens([3, 9, 4, 5]))  # the engine goes on as it was
    with pytest.raises(cuda_engine.QwenCudaError, match="outside vocabulary") as ei:
        own.logprobs([512])
    assert ei.value.code == cuda_engine.ERR_TOKEN
    with pytest.raises(cuda_engine.QwenCudaError, match="top must be"):
        own.logprobs([], 65)
    for b in (cuda_engine.Batch(eng, 3, 64), cuda_engine.Batch.paged(eng, 3, 64, BF16, 16, 12)):
        rows = b.forward([0, 2, 2], [5, 6, 7])
        ids = [[1, 2], [3, 511]]
        got = b.logprobs([2, 0], ids, 5)
        for i, row in enumerate((rows[1], rows[0])):
            check_logprobs(row, ids[i], 5, [a[i] for a in got])
        big = b.logprobs([0, 2, 0, 0, 2], None, 64)
        check_logprobs(rows[0], [], 64, [a[3] for a in big])
        with pytest.raises(cuda_engine.QwenCudaError, match="previous forward"):
            b.logprobs([1], [[0]])
        with pytest.raises(cuda_engine.QwenCudaError, match="sequence index"):
            b.logprobs([3], [[0]])


def test_engine_and_batches_go_in_any_order(cuda_engine, model):
    """Collected in one garbage cycle, or closed by hand, engine first."""
    import gc
    img, _, _ = model
    for close in (True, False):
        eng = cuda_engine.Engine(img, 32)
        some = [cuda_engine.Batch(eng, 2, 32), cuda_engine.Batch.paged(eng, 2, 32, F16, 16, 4, weights=True)]
        for b in some:
            b.forward([0, 1], [1, 2])
        if close:
            eng.close()
            for b in some:
                b.close()
        else:
            some.append(some)
            eng.cycle = some
            del eng, some, b
            gc.collect()
    eng = cuda_engine.Engine(img, 32)
    b = cuda_engine.Batch(eng, 1, 32)
    b.close()
    b.close()
    assert np.isfinite(eng.forward(1)).all()


def test_30b_shapes_in_pages(cuda_engine, tools):
    """Two layers of the 30B shapes: f32 pages against contiguous caches, bf16 pages with eviction at work
    (bf16 keys and values are off by up to 2^-8: as above, eight times that and the router's sharper turns)."""
    spec = tools.QWEN3_30B_A3B.with_(layers=2, vocab=2048)
    eng = cuda_engine.Engine(tools.synth_gguf(spec), 512)
    ps = prompts(spec, [200, 70, 131])
    seqs = [0] * 200 + [1] * 70 + [2] * 131
    a = cuda_engine.Batch(eng, 3, 512)
    b = cuda_engine.Batch.paged(eng, 3, 512, F32, 16, 40, weights=True)
    c = cuda_engine.Batch.paged(eng, 3, 512, BF16, 32, 24, weights=True)
    want = a.forward(seqs, sum(ps, []))
    got = b.forward(seqs, sum(ps, []))
    low = c.forward(seqs, sum(ps, []))
    scale = np.abs(want).max()
    assert np.abs(got - want).max() < 1e-3 * scale
    assert np.abs(low - want).max() < 0.1 * scale
    c.evict(64, 16)
    assert [c.cache(q)[0] for q in range(3)] == [64, 64, 64]
    for t in range(20):
        out = c.forward([0, 1, 2], [t, t, t])
        assert np.isfinite(out).all()
        if t % 8 == 7:
            c.evict(64, 16)
    assert [c.cache(q)[0] for q in range(3)] == [68, 68, 68]
    assert [c.position(q) for q in range(3)] == [220, 90, 151]
