"""Refusals of the paged cache's calls and of qc_logprobs that need no device: every argument that the
host can check is checked before CUDA is touched."""
import pytest

P = 1 << 20  # a well-aligned address that is never read


@pytest.fixture()
def E(cuda_engine):
    return cuda_engine


def cache(E, kind=1, k=P, v=P, n_pages=8, page=16, kvheads=2, head_dim=64, table=P, n_seqs=3, max_pages=4):
    return E.PagedCache(kind, k, v, n_pages, page, kvheads, head_dim, table, n_seqs, max_pages)


def refused(E, match, call, *a, **kw):
    with pytest.raises(E.QwenCudaError, match=match) as ei:
        call(*a, **kw)
    assert ei.value.code == E.ERR_INVALID


BAD = [
    (dict(kind=12), "F32, F16 or BF16"), (dict(kind=2), "F32, F16 or BF16"),
    (dict(k=None), "null argument"), (dict(table=None), "null argument"),
    (dict(n_pages=0), "empty cache"), (dict(page=0), "empty cache"), (dict(kvheads=0), "empty cache"),
    (dict(n_seqs=0), "empty cache"), (dict(max_pages=0), "empty cache"),
    (dict(head_dim=0), "multiple of 16 bytes"), (dict(head_dim=4), "multiple of 16 bytes"),
    (dict(head_dim=60), "multiple of 16 bytes"), (dict(head_dim=264), "multiple of 16 bytes"),
    (dict(kind=0, head_dim=6), "multiple of 16 bytes"),
    (dict(page=1 << 20, max_pages=1 << 12), "slots in a sequence"),
    (dict(n_pages=1 << 28, page=16), "rows in a pool"),
    (dict(kvheads=0xffffffff, head_dim=8), "rows in a pool"),
    (dict(n_seqs=0x7fffffff), "too many sequences"),
]


@pytest.mark.parametrize("bad,match", BAD)
def test_bad_caches_are_refused_by_every_call(E, bad, match):
    c = cache(E, **bad)
    refused(E, match, c.append, P, P, 1, P)
    refused(E, match, c.attention, P, bad.get("kvheads", 2) or 2, 1, P, P)
    refused(E, match, c.evict, P, P, 8, 2, P, P)


def test_bad_calls_are_refused(E):
    c = cache(E)
    refused(E, "null argument", c.append, None, P, 1, P)
    refused(E, "null argument", c.append, P, P, 1, None)
    refused(E, "more rows than sequences", c.append, P, P, 4, P)
    refused(E, "heads must be", c.attention, P, 3, 1, P, P)
    refused(E, "heads must be", c.attention, P, 0, 1, P, P)
    refused(E, "heads must be", c.attention, P, 66, 1, P, P)
    refused(E, "scale", c.attention, P, 4, 1, P, P, scale=float("nan"))
    refused(E, "scale", c.attention, P, 4, 1, P, P, scale=float("inf"))
    refused(E, "null argument", c.attention, None, 4, 1, P, P)
    refused(E, "null argument", c.attention, P, 4, 1, None, P)
    refused(E, "null argument", c.attention, P, 4, 1, P, None)
    refused(E, "more rows than sequences", c.attention, P, 4, 4, P, P)
    refused(E, "weights need lse", c.attention, P, 4, 1, P, P, weights_ptr=P)
    refused(E, "8192 sequences", cache(E, n_seqs=8193).attention, P, 4, 2, P, P, seq_ptr=P, lse_ptr=P, weights_ptr=P)
    refused(E, "too many rows", c.attention, P, 4, 0xffffffff, P, P, seq_ptr=P)
    refused(E, "keep must be", c.evict, P, P, 0, 0, P, P)
    refused(E, "keep must be", c.evict, P, P, 65, 0, P, P)
    refused(E, "recent must be", c.evict, P, P, 8, 9, P, P)
    refused(E, "null argument", c.evict, P, None, 8, 2, P, P)
    refused(E, "null argument", c.evict, P, P, 8, 2, None, P)
    # alignment is checked before the device is asked
    refused(E, "k_pages is not 16-byte aligned", cache(E, k=P + 8).append, P, P, 1, P)
    # no rows: nothing to do, whatever the pointers
    c.append(None, None, 0, None)
    c.attention(None, 4, 0, None, None)


def test_bad_logprobs_are_refused(E):
    refused(E, "empty logits", E.logprobs, P, 1, 0)
    refused(E, "top must be", E.logprobs, P, 1, 100, top=65, top_ids_ptr=P, top_logprobs_ptr=P)
    refused(E, "top must be", E.logprobs, P, 1, 3, top=4, top_ids_ptr=P, top_logprobs_ptr=P)
    refused(E, "null argument", E.logprobs, P, 1, 100, top=4, top_ids_ptr=P)
    refused(E, "null argument", E.logprobs, P, 1, 100, n_ids=1, ids_ptr=P)
    refused(E, "null argument", E.logprobs, P, 1, 100, n_ids=1, logprobs_ptr=P)
    refused(E, "null argument", E.logprobs, None, 1, 100)
    refused(E, "rows overlap", E.logprobs, P, 2, 100, stride=99)
    refused(E, "too many logits", E.logprobs, P, 1, 0x80000000)
    refused(E, "logits is not 4-byte aligned", E.logprobs, P + 2, 1, 100)
    E.logprobs(None, 0, 100)
