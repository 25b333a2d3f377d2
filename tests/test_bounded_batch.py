"""Eviction in batches (qc_batch_evict) against the same model in 64 bits, its caches held to the same budget."""
import numpy as np
import pytest

from _bounded import Bounded

F32 = 0
# what is done: tokens fed, then an eviction (keep, recent) of sequence 0
PLAN = [(70, 30, 6), (9, 24, 0), (17, 33, 20), (12, 25, 24), (8, 30, 30), (10, 0, 0)]


def spec_of(tools):
    return tools.TINY.with_(layers=3)


def tokens_of(spec):
    return np.random.default_rng(42).integers(0, spec.vocab, sum(n for n, _, _ in PLAN)).tolist()


def run(model, tokens):
    """The logits after every token but the first sixty, and the cached slots after each eviction."""
    at, rows, sizes = 0, [], []
    for n, keep, recent in PLAN:
        for t in tokens[at:at + n]:
            row = model.forward(t)
            if model.position > 60:
                rows.append(row)
        at += n
        if keep:
            model.evict(keep, recent)
            sizes.append(len(model.slots[0][0]["w"]))
    return np.stack(rows), sizes


@pytest.fixture(scope="module")
def expected(tools, oracle):
    spec = spec_of(tools)
    img = tools.synth_gguf(spec)
    model = Bounded(img, spec, oracle)
    rows, sizes = run(model, tokens_of(spec))
    # (f32 sums of some hundred terms are off by 1e-6 to 1e-5: no choice hangs on that)
    assert model.margin > 5e-4, model.margin
    return spec, img, rows, sizes


def test_the_plain_model_is_the_oracles(expected, oracle):
    spec, img, _, _ = expected
    plain, ref = Bounded(img, spec, oracle), oracle.Model(img, 256)
    for t in tokens_of(spec)[:40]:
        assert np.abs(plain.forward(t) - ref.forward(t)).max() < 1e-4


@pytest.mark.parametrize("wrong", ["layer 0", "smallest", "no recent", "one head's slots", "weights stay"])
def test_mistakes_would_show(expected, oracle, wrong):
    spec, img, rows, sizes = expected
    other, n = run(Bounded(img, spec, oracle, wrong), tokens_of(spec))
    assert n == sizes
    assert np.abs(other - rows).max() > 2e-2, np.abs(other - rows).max()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("whole", [False, True])
def test_a_batch_keeps_what_the_plain_model_keeps(cuda_engine, oracle, expected, page, whole):
    """Sequence 1 of three is held to the budget; the others go on undisturbed.  Logits within the decode path's
    1e-3.  whole: every stretch of tokens as one call, which gives its last row only."""
    spec, img, rows, sizes = expected
    eng = cuda_engine.Engine(img, 256)
    b = cuda_engine.Batch.paged(eng, 3, 256, F32, page, 3 * 60, weights=True)
    tokens, at, got, where = tokens_of(spec), 0, [], []
    other = oracle.Model(img, 256)
    side, first = [], None
    for t in tokens[:50]:
        first = other.forward(t)
    for k, (n, keep, recent) in enumerate(PLAN):
        if k == 1:  # another sequence joins
            assert np.abs(b.forward([2] * 50, tokens[:50])[0] - first).max() < 1e-3
        stretch = tokens[at:at + n]
        if whole:
            got.append(b.forward([1] * n, stretch)[0])
            where.append(at + n - 61)
        else:
            for i, t in enumerate(stretch):
                row = b.forward([1], [t])[0]
                if at + i >= 60:
                    got.append(row)
                    where.append(at + i - 60)
        at += n
        if keep:
            b.evict(keep, recent, seq=1)
            assert b.cache(1)[0] == sizes[k] and b.position(1) == at
        if k:
            side.append((b.forward([2], [k])[0], other.forward(k)))
    err = np.abs(np.stack(got) - rows[where]).max(1)
    assert err.max() < 1e-3, (where[int(err.argmax())], err.max())
    assert all(np.abs(a - w).max() < 1e-3 for a, w in side)
