"""Paged attention where keys or values are as large as their type allows.

Bounds are attention64's: a slot without weight adds nothing to them."""
import math

import pytest
import torch

from _paged import DTYPE, Cache, attention64, ptr

pytestmark = pytest.mark.gpu

SHARED = [1, 32]  # rows of a sequence: by themselves, and together (16 rows a sequence and more)


def run(E, cache, q, seq, lens, weights=None):
    sq, ln = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, lens))
    out = torch.full(q.shape, 7.0, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    cache.handle(E).attention(ptr(q), q.shape[1], len(lens), ptr(ln), ptr(out), seq_ptr=ptr(sq), lse_ptr=ptr(lse),
                              weights_ptr=ptr(weights))
    torch.cuda.synchronize()
    return out, lse


def put(cache, pool, s, j, value):
    """value: of slot j of sequence s, all KV heads."""
    getattr(cache, pool)[int(cache.table[s, j // cache.page]), :, j % cache.page] = value


def without(cache, hidden):
    """Sequence 0 without its first `hidden` slots, as a cache of its own."""
    n = cache.lens[0] - hidden
    rest = Cache(cache.kind, cache.kvheads, cache.D, cache.page, [n])
    for pool in "kv":
        rows = cache.rows(0, cache.lens[0], pool)[hidden:]
        for j in range(n):
            put(rest, pool, 0, j, rows[j])
    return rest


def check_hidden(E, cache, q, hidden, rows):
    """The first `hidden` slots have no weight; a row that sees only them sees nothing."""
    n = cache.lens[0]
    seq, lens = [0] * rows, [n] * rows
    if rows > 1:
        lens[1], lens[rows - 1] = hidden, n - 1
    weights = torch.zeros(1, cache.kvheads, cache.cap, device="cuda")
    out, lse = run(E, cache, q, seq, lens, weights)
    rest = without(cache, hidden)
    seen = [i for i in range(rows) if lens[i] > hidden]
    want, wlse, _, eo, _ = attention64(rest, q[seen], [0] * len(seen), [lens[i] - hidden for i in seen], 1 / math.sqrt(cache.D))
    for k, i in enumerate(seen):
        assert bool(((out[i].double() - want[k]).abs() <= eo[k]).all()), i
        assert torch.allclose(lse[i].double(), wlse[k], rtol=2e-6, atol=2e-5), i
    for i in set(range(rows)) - set(seen):
        assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())
    assert bool((weights[..., :hidden] == 0).all()) and bool(weights[..., :n].isfinite().all())


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("D,page", [(64, 16), (96, 5), (128, 16), (256, 24)])
def test_f32_keys_of_the_lowest_value_have_no_weight(cuda_engine, torch_cuda, D, page, rows):
    """-FLT_MAX and what rounds to it, against queries with zeros among their values."""
    cache = Cache("f32", 2, D, page, [50], seed=D)
    lowest = -torch.finfo(torch.float32).max
    for j in range(7):
        put(cache, "k", 0, j, lowest * (1 - j * 2.0 ** -14))
    q = torch.full((rows, 8, D), 4.0, device="cuda")
    q[:, :, 1::3] = 0
    check_hidden(cuda_engine, cache, q, 7, rows)


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,page", [(64, 16), (96, 5), (256, 24)])
def test_values_of_the_largest_size(cuda_engine, torch_cuda, kind, D, page, rows):
    cache = Cache(kind, 2, D, page, [50], seed=D)
    most = torch.finfo(DTYPE[kind]).max
    value = cache.rows(0, 50, "v")[3].clone()
    value[:, 5], value[:, 6], value[:, 7] = most, -most, most * (1 - 2.0 ** -8)
    put(cache, "v", 0, 3, value)
    q = torch.randn(rows, 8, D, generator=torch.Generator().manual_seed(1)).cuda()
    lens = [50 - i % 3 for i in range(rows)]
    out, _ = run(cuda_engine, cache, q, [0] * rows, lens)
    want, _, _, eo, _ = attention64(cache, q, [0] * rows, lens, 1 / math.sqrt(D))
    for i in range(rows):
        assert bool(out[i].isfinite().all()) and bool(((out[i].double() - want[i]).abs() <= eo[i]).all()), i


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D,size", [(64, 4.0), (64, 155.0), (64, 1418.0), (128, 155.0), (128, 3999.0), (32, 30000.0)])
def test_keys_of_the_lowest_value_have_no_weight(cuda_engine, torch_cuda, kind, D, size, rows):
    """Queries of one size, whose roundings to the pages' type add up, in either direction.  (The lowest f16 number
    gives a finite score: the next test.)"""
    cache = Cache(kind, 2, D, 16, [50], seed=D)
    for j in range(7):
        put(cache, "k", 0, j, -torch.finfo(DTYPE[kind]).max)
    for j in range(7, 50):  # scores of the others of an ordinary size
        put(cache, "k", 0, j, cache.rows(0, 50)[j] * (4.0 / size))
    q = torch.full((rows, 8, D), size, device="cuda")
    q[:, 4:, 1::3] = 0
    check_hidden(cuda_engine, cache, q, 7, rows)


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("size", [4.0, 155.0, 30000.0])
def test_f16_keys_of_the_lowest_value(cuda_engine, torch_cuda, size, rows):
    """Their scores are finite: no weight beside others (exp underflows), equal weights among themselves."""
    cache = Cache("f16", 2, 64, 16, [50], seed=2)
    for j in range(7):
        put(cache, "k", 0, j, -torch.finfo(torch.float16).max)
    q = torch.full((rows, 8, 64), size, device="cuda")
    q[:, 4:, 1::3] = 0
    lens = [50 if i % 2 == 0 else 7 for i in range(rows)]
    out, lse = run(cuda_engine, cache, q, [0] * rows, lens)
    want, wlse, _, eo, _ = attention64(cache, q, [0] * rows, lens, 0.125)
    rest, rlse, _, er, _ = attention64(without(cache, 7), q, [0] * rows, [43] * rows, 0.125)
    for i in range(rows):
        w, l, e = (rest[i], rlse[i], er[i]) if lens[i] == 50 else (want[i], wlse[i], eo[i])
        assert bool(((out[i].double() - w).abs() <= e).all()), i
        assert torch.allclose(lse[i].double(), l, rtol=2e-6, atol=2e-5), i
        assert torch.allclose(w, want[i], rtol=1e-12, atol=1e-12)  # (the formula says the same)


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_infinite_keys_count_as_their_scores_say(cuda_engine, torch_cuda, kind, rows):
    """-inf in one value of a key: a score of -inf for queries that are positive there, +inf for negative ones, NaN
    for zeros; the last two leave no softmax."""
    cache = Cache(kind, 1, 64, 16, [50], seed=3)
    for j in range(3):
        key = cache.rows(0, 50)[j].clone()
        key[:, 9] = -math.inf
        put(cache, "k", 0, j, key)
    q = torch.randn(rows, 8, 64, generator=torch.Generator().manual_seed(1)).cuda()
    q[:, :, 9] = torch.tensor([0.5, 1.0, 0.3, 77.7, 1.1, -0.5, 0.0, -3.3], device="cuda")
    out, lse = run(cuda_engine, cache, q, [0] * rows, [50] * rows)
    rest = without(cache, 3)
    want, wlse, _, eo, _ = attention64(rest, q, [0] * rows, [47] * rows, 0.125)
    for i in range(rows):
        assert bool(((out[i, :5].double() - want[i][:5]).abs() <= eo[i][:5]).all())
        assert torch.allclose(lse[i, :5].double(), wlse[i][:5], rtol=2e-6, atol=2e-5)
        assert not bool(out[i, 5:].isfinite().any())


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0x7FC00000, 0x7FFFFFFF, 0x7F800001, 0xFFFFFFFF])
def test_nan_is_never_lost(cuda_engine, torch_cuda, kind, bits, rows):
    """A NaN key beside one of the lowest value in the same row, and NaN among the queries, leave no softmax."""
    nan = torch.tensor([bits - (1 << 32 if bits >> 31 else 0)], dtype=torch.int32).view(torch.float32)
    cache = Cache(kind, 1, 64, 16, [50], seed=3)
    key = cache.rows(0, 50)[4].clone()
    if kind == "f32":
        key.view(torch.int32)[:, 9] = nan.view(torch.int32).cuda()
    else:
        key[:, 9] = math.nan
    key[:, 11:40] = -torch.finfo(DTYPE[kind]).max
    put(cache, "k", 0, 4, key)
    q = torch.full((rows, 8, 64), 300.0, device="cuda")
    out, lse = run(cuda_engine, cache, q, [0] * rows, [50] * rows)
    assert not bool(out.isfinite().any()) and not bool(lse.isfinite().any())
    put(cache, "k", 0, 4, torch.full_like(key, -torch.finfo(DTYPE[kind]).max))
    q.view(torch.int32)[:, 2, 5] = nan.view(torch.int32).cuda()
    out, lse = run(cuda_engine, cache, q, [0] * rows, [50] * rows)
    assert not bool(out[:, 2].isfinite().any()) and not bool(lse[:, 2].isfinite().any())
    assert bool(out[:, [0, 1, 3, 4, 5, 6, 7]].isfinite().all())


@pytest.mark.parametrize("rows", SHARED)
@pytest.mark.parametrize("D", [96, 128, 192, 256])
def test_f32_scores_are_not_cut_in_one_long_sum(cuda_engine, torch_cuda, D, rows):
    """Products of one sign, whose sum the matrix units cut towards zero at every step of eight: the sum so far and
    the step's eight products each by half a last place on average, at most 2^-24 of the sum.  m equal steps lose
    m + 1 of those of their whole sum; rows by themselves have four sums of D / 32 steps, rows together two of D / 16.
    lse is s + log n here, with s far larger; its own roundings, and those of queries and keys, are to the nearest and
    vanish in the mean: 1.5 for what is left."""
    n, heads = 100, 8
    cache = Cache("f32", 2, D, 16, [n], seed=D)
    g = torch.Generator().manual_seed(D)
    for j in range(n):
        put(cache, "k", 0, j, (0.5 + torch.rand(2, D, generator=g)).cuda())
    q = 16 * (0.5 + torch.rand(rows if rows > 1 else 24, heads, D, generator=g)).cuda()
    if rows > 1:
        _, lse = run(cuda_engine, cache, q, [0] * rows, [n] * rows)
    else:
        lse = torch.cat([run(cuda_engine, cache, q[i:i + 1].contiguous(), [0], [n])[1] for i in range(24)])
    _, want, _, _, _ = attention64(cache, q, [0] * len(q), [n] * len(q), 1 / math.sqrt(D))
    want = torch.stack(want)
    bias = float(((lse.double() - want) / want).mean()) / 2.0 ** -24
    steps = D / (32 if rows == 1 else 16)
    assert abs(bias) <= steps + 1 + 1.5, bias
