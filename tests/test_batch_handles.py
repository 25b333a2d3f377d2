"""Handles of batches whose engine is gone: every call is refused, none reaches the freed batch.  (The
library's destructors are stood in for: no device is needed.)"""
import ctypes

import pytest


class Library:
    """The library, with engines and batches that are only numbers."""

    def __init__(self, real):
        self.real, self.destroyed = real, []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def qc_batch_destroy(self, h):
        if h.value:
            self.destroyed.append(("batch", h.value))

    def qc_engine_destroy(self, h):
        self.destroyed.append(("engine", h.value))


@pytest.fixture()
def made(cuda_engine, monkeypatch):
    E = cuda_engine
    library = Library(E.lib())
    monkeypatch.setattr(E, "lib", lambda: library)
    eng = E.Engine.__new__(E.Engine)
    eng._h, eng.vocab = ctypes.c_void_p(0x1000), 16
    batches = []
    for address in (0x2000, 0x3000):
        b = E.Batch.__new__(E.Batch)
        b._h, b.engine, b.n_seqs, b.context, b.vocab = ctypes.c_void_p(address), eng, 2, 32, 16
        eng._adopt(b._h)
        batches.append(b)
    return E, library, eng, batches


def calls(E, b):
    smp = E.Sampler.__new__(E.Sampler)
    smp._h = None
    return [lambda: b.forward([0], [1]), lambda: b.logprobs([0], [[1]], 2), lambda: b.cache(0), lambda: b.evict(4, 1),
            lambda: b.reset(), lambda: b.position(0), lambda: b.logits_device_ptr(0), lambda: b.sample([], [0]),
            lambda: b.decode_sample([], [0], 1), lambda: b.stats(), lambda: b.ep_handle(),
            lambda: b.connect([(bytes(64), 0)])]


def test_calls_after_the_engine_is_closed_are_refused(made):
    E, library, eng, batches = made
    eng.close()
    assert library.destroyed == [("batch", 0x2000), ("batch", 0x3000), ("engine", 0x1000)]
    for b in batches:
        for call in calls(E, b):
            with pytest.raises(E.QwenCudaError, match="null batch") as ei:
                call()
            assert ei.value.code == E.ERR_INVALID
        b.close()
        b.close()
    eng.close()
    assert len(library.destroyed) == 3


def test_a_closed_batch_is_not_destroyed_again(made):
    E, library, eng, batches = made
    batches[0].close()
    assert library.destroyed == [("batch", 0x2000)]
    for call in calls(E, batches[0]):
        # (the engine is only a number, and the message is asked of it: the code is not)
        eng._h = None
        with pytest.raises(E.QwenCudaError, match="null batch"):
            call()
    eng._h = ctypes.c_void_p(0x1000)
    eng.close()
    assert library.destroyed == [("batch", 0x2000), ("batch", 0x3000), ("engine", 0x1000)]
    batches[0].close(), batches[1].close()
    assert len(library.destroyed) == 3


@pytest.mark.gpu
def test_an_engine_closed_under_its_batches(cuda_engine, tools):
    with cuda_engine.Engine(tools.synth_gguf(tools.TINY), 32) as eng:
        batches = [cuda_engine.Batch(eng, 2, 32),
                   cuda_engine.Batch.paged(eng, 2, 32, cuda_engine.PagedCache.F16, 16, 4, weights=True)]
        for b in batches:
            b.forward([0, 1], [1, 2])
    for b in batches:
        for call in (lambda: b.forward([0], [1]), lambda: b.logprobs([0], [[1]], 2), lambda: b.evict(4, 1)):
            with pytest.raises(cuda_engine.QwenCudaError, match="null batch"):
                call()
        b.close()


def test_log_probabilities_of_no_sequence_are_refused(made):
    """By the library, as every bad call (here the batch is gone as well)."""
    E, _, eng, batches = made
    eng.close()
    for ids in (None, [], [[]], [[1, 2]]):
        with pytest.raises(E.QwenCudaError):
            batches[0].logprobs([], ids, 2)


@pytest.mark.gpu
def test_log_probabilities_of_no_sequence(cuda_engine, tools):
    eng = cuda_engine.Engine(tools.synth_gguf(tools.TINY), 32)
    b = cuda_engine.Batch(eng, 2, 32)
    b.forward([0, 1], [1, 2])
    for ids in (None, [], [[]]):
        with pytest.raises(cuda_engine.QwenCudaError, match="empty batch"):
            b.logprobs([], ids, 2)
    assert b.logprobs([1, 0], [[3], [4]])[0].shape == (2, 1) and b.logprobs([1, 0], [3, 4])[0].shape == (2, 1)
