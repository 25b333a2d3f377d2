"""Eviction in place where sequences, or the first of their slots, stay where they are."""
import pytest
import torch

from _paged import Cache, evict64, ptr

pytestmark = pytest.mark.gpu


def evict(E, cache, weights, lens, keep, recent, dst=None, new=None, wout=None):
    S = len(cache.lens)
    kept = torch.zeros(S, cache.kvheads, keep, dtype=torch.int32, device="cuda")
    new = lens if new is None else new
    cache.handle(E).evict(ptr(weights), ptr(lens), keep, recent, ptr(kept), ptr(new), weights_out_ptr=ptr(wout),
                          dst_table_ptr=ptr(dst))
    return kept, new


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,keep", [(2, 1), (200, 128), (300, 255), (300, 256), (300, 257), (1000, 513), (5000, 4097),
                                    (70100, 70001)])
def test_slots_before_the_first_that_goes_stay(cuda_engine, torch_cuda, kind, n, keep):
    """The lightest slots begin at a given one: nothing before it moves."""
    firsts = sorted({0, 1, 2, keep // 256, keep // 256 + 1, 127, 128, 129, keep // 2, keep - 2, keep - 1, keep} - {-1})
    firsts = [f for f in firsts if 0 <= f <= keep and f + (n - keep) <= n]
    # one sequence for each first slot that goes, one within the budget, an empty one
    lens = [n] * len(firsts) + [keep, max(1, keep - 1), 0]
    cache = Cache(kind, 2, 8, 16, lens, seed=keep)
    w = 1 + torch.rand(len(lens), 2, cache.cap, generator=torch.Generator().manual_seed(n))
    for s, f in enumerate(firsts):
        w[s, :, f:f + n - keep] = 0.5
        w[s, 1, f] = 3.0  # the other KV head: a slot further
        if f + n - keep < n:
            w[s, 1, f + n - keep] = 0.25
    weights, lens_d = w.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    old = {p: [cache.rows(s, m, p).clone() for s, m in enumerate(lens)] for p in "kv"}
    kept, new = evict(cuda_engine, cache, weights, lens_d, keep, 0)
    torch.cuda.synchronize()
    assert new.tolist() == [min(m, keep) for m in lens]
    for s, length in enumerate(lens):
        m = min(length, keep)
        for h in range(2):
            want = evict64(w[s, h], length, keep, 0)
            assert kept[s, h].tolist() == want + [-1] * (keep - m)
            assert torch.equal(weights[s, h, :m].cpu(), w[s, h][want])
            for p in "kv":
                assert torch.equal(cache.rows(s, m, p)[:, h], old[p][s][want, h]), (s, h, p)
    for s, f in enumerate(firsts):
        assert kept[s, 0, :f].tolist() == list(range(f))


def test_sequences_within_their_budget_are_not_copied(cuda_engine, torch_cuda):
    """1 GB of rows that stay take no longer than reading their weights' order; to other pages they are copied."""
    S, n, keep = 64, 4000, 4096
    cache = Cache("bf16", 4, 128, 16, [n] * S, spare=S * 250, seed=1)
    free = sorted(set(range(cache.n_pages)) - set(cache.table.flatten().tolist()))
    dst = torch.tensor(free[: S * cache.max_pages], dtype=torch.int32).reshape(S, -1).cuda()
    weights = torch.rand(S, 4, cache.cap, device="cuda")
    wout, lens = torch.zeros_like(weights), torch.tensor(cache.lens, dtype=torch.int32, device="cuda")
    new = torch.zeros_like(lens)
    keep = min(keep, cache.cap)

    def us(**to):
        best = 1e30
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            for _ in range(4):
                evict(cuda_engine, cache, weights, lens, keep, 10, new=new, **to)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) / 4 * 1e3)
        return best

    before = cache.k.clone()
    us()
    elsewhere, in_place = us(dst=dst, wout=wout), us()
    assert torch.equal(cache.rows(5, n).view(torch.int16), before[cache.table[5].long()[torch.arange(n, device="cuda") // 16], :,
                                                                  torch.arange(n, device="cuda") % 16].view(torch.int16))
    assert in_place < elsewhere / 3, (in_place, elsewhere)
