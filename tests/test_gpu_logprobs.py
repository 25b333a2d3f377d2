"""qc_logprobs against log-softmax in 64 bits.

Bounds: d = x - max is rounded once, 2^-24 |d|; the sum's terms carry exp's 2 ulp and the rounding of d
times log2 e, 2^-24 |d|, each its own, so that the sum is good to about 1e-6 with the few hundred
additions in a row that a lane makes.  A log probability is held to 2^-21 |d| + 2e-6 of it, or of one
where it is larger; the entropy to 5e-6 of it.
"""
import math

import pytest
import torch

from _paged import ptr

pytestmark = pytest.mark.gpu


def run(E, x, ids=None, top=0, entropy=True, stride=None, n=None, rows=None, stream=None):
    rows, n = rows or x.shape[0], n or x.shape[1]
    n_ids = ids.shape[1] if ids is not None else 0
    lp = torch.full((rows, max(1, n_ids)), 9.0, device="cuda")
    ent = torch.full((rows,), 9.0, device="cuda")
    ti = torch.full((rows, max(1, top)), 9, dtype=torch.int32, device="cuda")
    tl = torch.full((rows, max(1, top)), 9.0, device="cuda")
    E.logprobs(x.data_ptr(), rows, n, stride=stride, ids_ptr=ptr(ids), n_ids=n_ids, top=top, logprobs_ptr=ptr(lp),
               entropy_ptr=ptr(ent) if entropy else None, top_ids_ptr=ptr(ti), top_logprobs_ptr=ptr(tl), stream=stream)
    torch.cuda.synchronize()
    return lp[:, :n_ids], ent, ti[:, :top], tl[:, :top]


def check(x, ids, top, got):
    lp, ent, ti, tl = got
    xd = x.double()
    m = xd.amax(-1, keepdim=True)
    want = xd - torch.logsumexp(xd, -1, keepdim=True)
    err = 2.0 ** -21 * (xd - m).abs().clamp(max=1e30) + 2e-6 * want.abs().clamp(max=1)
    if ids is not None:
        w, e = want.gather(-1, ids.long()), err.gather(-1, ids.long())
        assert bool(((lp.double() - w).abs() <= e)[w.isfinite()].all()), float((lp.double() - w)[w.isfinite()].abs().max())
        assert bool((lp[~w.isfinite()] == -math.inf).all())
    p = want.exp()
    h = -(p * torch.where(p > 0, want, 0.0)).sum(-1)
    assert bool(((ent.double() - h).abs() <= 4e-6 * h + 1e-6 * torch.minimum(h, torch.ones_like(h)) + 1e-30).all()), \
        float((ent.double() - h).abs().max())
    order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ti.long(), order)
    w, e = want.gather(-1, order), err.gather(-1, order)
    assert bool(((tl.double() - w).abs() <= e)[w.isfinite()].all())
    assert bool((tl[~w.isfinite()] == -math.inf).all())


SIZES = [(1, 1, 1, 1), (3, 2, 2, 2), (2, 5, 3, 0), (7, 63, 1, 63), (5, 64, 0, 64), (4, 257, 9, 17), (1, 1000, 1, 1),
         (9, 4097, 2, 64), (33, 8191, 1, 5), (2, 50257, 4, 20), (1, 151936, 1, 20), (40, 151936, 1, 64),
         (300, 32003, 1, 3), (2, 700001, 2, 64), (1, 2500000, 1, 7)]


@pytest.mark.parametrize("rows,n,n_ids,top", SIZES)
@pytest.mark.parametrize("scale", [0.3, 4.0])
def test_logprobs_match_the_formula(cuda_engine, torch_cuda, rows, n, n_ids, top, scale):
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(rows, n, generator=g) * scale).cuda()
    ids = torch.randint(0, n, (rows, n_ids), generator=g, dtype=torch.int32).cuda() if n_ids else None
    got = run(cuda_engine, x, ids, top)
    check(x, ids, top, got)
    again = run(cuda_engine, x, ids, top)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("rows,n,top", [(3, 1000, 64), (2, 151936, 64), (1, 700001, 64), (150, 9001, 20)])
@pytest.mark.parametrize("values", ["equal", "few", "rising", "falling", "masked", "peaked"])
def test_hard_orders(cuda_engine, torch_cuda, rows, n, top, values):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, n, generator=g)
    if values == "equal":
        x = torch.full_like(x, -2.5)
    elif values == "few":
        x = torch.floor(x * 1.5)
        x = torch.where(x == 0, torch.where(torch.rand(x.shape, generator=g) < 0.5, 0.0, -0.0), x)
    elif values == "rising":
        x = torch.arange(n).float().expand(rows, n) * 1e-3
    elif values == "falling":
        x = torch.arange(n, 0, -1).float().expand(rows, n) * 1e-3
    elif values == "masked":  # most ids masked, by -inf and by the type's lowest value
        hide = torch.rand(rows, n, generator=g)
        x = torch.where(hide < 0.7, -math.inf, torch.where(hide < 0.95, torch.finfo(torch.float32).min, x))
        x[:, n // 2] = 1.0
    else:  # one id nearly certain: log p close to 0
        x[:, n // 3] = 25.0
    x = x.contiguous().cuda()
    ids = torch.stack([torch.full((rows,), i) for i in (0, n // 3, n // 2, n - 1)], 1).to(torch.int32).cuda()
    check(x, ids, top, run(cuda_engine, x, ids, top))


def test_strides_alignment_and_what_is_left(cuda_engine, torch_cuda):
    g = torch.Generator().manual_seed(1)
    for n, stride, shift in [(1003, 1007, 1), (151936, 151939, 3), (64, 101, 2), (9001, 9001, 1)]:
        buf = torch.full((5 * stride + 8,), math.nan)
        for r in range(5):
            buf[shift + r * stride: shift + r * stride + n] = torch.randn(n, generator=g) * 2
        buf = buf.cuda()
        x = torch.stack([buf[shift + r * stride: shift + r * stride + n] for r in range(5)])
        ids = torch.randint(0, n, (5, 2), generator=g, dtype=torch.int32).cuda()
        check(x, ids, 11, run(cuda_engine, buf[shift:], ids, 11, stride=stride, n=n, rows=5))
    # nothing asked for is nothing written
    x = torch.randn(2, 100, generator=g).cuda()
    lp, ent, ti, tl = run(cuda_engine, x, None, 0, entropy=False)
    assert bool((ent == 9).all()) and lp.numel() == 0 and ti.numel() == 0


@pytest.mark.parametrize("n", [5, 3001, 151936])
def test_rows_without_a_distribution(cuda_engine, torch_cuda, n):
    x = torch.randn(5, n, generator=torch.Generator().manual_seed(2))
    x[1, n // 2] = math.nan
    x[2, n - 1] = math.inf
    x[3] = -math.inf
    x = x.cuda()
    ids = torch.tensor([[0, 1, n], [0, 1, 2], [0, 1, 2], [0, 1, 2], [2, -1, 1]], dtype=torch.int32).cuda()
    lp, ent, ti, tl = run(cuda_engine, x, ids, 4)
    good = run(cuda_engine, x[[0, 4]].contiguous(), ids[[0, 4]].contiguous(), 4)
    assert torch.equal(lp[[0, 4]].nan_to_num(5), good[0].nan_to_num(5))
    assert bool(lp[0, 2].isnan()) and bool(lp[4, 1].isnan()) and int(lp[[0, 4]].isnan().sum()) == 2  # ids out of range
    for r in (1, 2, 3):
        assert bool(lp[r].isnan().all()) and bool(ent[r].isnan()) and bool(tl[r].isnan().all())
    order = torch.sort(torch.where(x[1].isnan(), -math.inf, x[1]), descending=True, stable=True).indices[:4]
    assert torch.equal(ti[1].long(), order)
    assert int(ti[2, 0]) == n - 1 and ti[3].tolist() == [0, 1, 2, 3]


def test_captured_and_on_another_stream(cuda_engine, torch_cuda):
    x = torch.randn(6, 40000, device="cuda")
    ids = torch.randint(0, 40000, (6, 1), dtype=torch.int32, device="cuda")
    out = [torch.zeros(6, 1, device="cuda"), torch.zeros(6, device="cuda"),
           torch.zeros(6, 8, dtype=torch.int32, device="cuda"), torch.zeros(6, 8, device="cuda")]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cuda_engine.logprobs(ptr(x), 6, 40000, ids_ptr=ptr(ids), n_ids=1, top=8, logprobs_ptr=ptr(out[0]),
                             entropy_ptr=ptr(out[1]), top_ids_ptr=ptr(out[2]), top_logprobs_ptr=ptr(out[3]),
                             stream=torch.cuda.current_stream().cuda_stream)
    for seed in range(2):
        x.copy_(torch.randn(6, 40000, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        want = run(cuda_engine, x, ids, 8)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
