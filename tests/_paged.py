"""Plain 64-bit forms of the paged cache's operators and the device data they run on."""
import torch

KIND = {"f32": 0, "f16": 1, "bf16": 30}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """Pools of random pages; every slot that no sequence has cached holds NaN."""

    def __init__(self, kind, kvheads, D, page, lens, cap=None, spare=3, seed=0, n_pages=None):
        self.kind, self.kvheads, self.D, self.page, self.lens = kind, kvheads, D, page, list(lens)
        S = len(lens)
        self.max_pages = max(1, -(-max([cap or 1, *lens]) // page))
        self.cap = self.max_pages * page
        g = torch.Generator().manual_seed(seed)
        self.n_pages = n_pages or S * self.max_pages + spare
        perm = torch.randperm(self.n_pages, generator=g)[: S * self.max_pages].reshape(S, self.max_pages)
        self.table = perm.to(torch.int32).cuda()
        self.k = torch.full((self.n_pages, kvheads, page, D), float("nan"), dtype=DTYPE[kind], device="cuda")
        self.v = self.k.clone()
        for s, n in enumerate(self.lens):
            for pool in (self.k, self.v):
                rows = torch.randn(n, kvheads, D, generator=g).to(DTYPE[kind]).cuda()
                at = torch.arange(n, device="cuda")
                pool[self.table[s].long()[at // page], :, at % page] = rows

    def handle(self, E):
        return E.PagedCache(KIND[self.kind], ptr(self.k), ptr(self.v), self.n_pages, self.page, self.kvheads, self.D,
                            ptr(self.table), len(self.lens), self.max_pages)

    def rows(self, s, n, which="k", table=None):
        """Slots 0..n-1 of sequence s: [n][kvheads][D] in the cache's type."""
        at = torch.arange(n, device="cuda")
        t = (self.table if table is None else table)[s].long()
        return getattr(self, which)[t[at // self.page], :, at % self.page]


def attention64(cache, q, seq, lens, scale):
    """(out, lse, per-row weights) of the formula in 64 bits, and the bounds of an f32 computation.

    Scores: a sum of D products in f32, each addition off by at most 2^-23 of the running sum (the
    matrix units truncate), operands exact to 2^-21:  es = (D + 8) 2^-23 scale sum |q k|.
    exp(s - lse) is then off by 2 es + 2^-20 relatively (both s and lse carry es; exp, the joins of the
    splits).  The sums over positions add at most 2^-23 an addition, over n / 4 additions in a row."""
    outs, lses, ws, eo, ew = [], [], [], [], []
    heads, D = q.shape[1:]
    G = heads // cache.kvheads
    for i, (s, n) in enumerate(zip(seq, lens)):
        if n == 0:
            outs.append(torch.zeros(heads, D, dtype=torch.float64, device="cuda"))
            lses.append(torch.full((heads,), -float("inf"), dtype=torch.float64, device="cuda"))
            ws.append(torch.zeros(cache.kvheads, 0, dtype=torch.float64, device="cuda"))
            eo.append(torch.zeros(heads, D, dtype=torch.float64, device="cuda"))
            ew.append(torch.zeros(cache.kvheads, 0, dtype=torch.float64, device="cuda"))
            continue
        k = cache.rows(s, n, "k").double().repeat_interleave(G, 1)
        v = cache.rows(s, n, "v").double().repeat_interleave(G, 1)
        qd = q[i].double()
        sc = torch.einsum("hd,nhd->hn", qd, k) * scale
        es = ((D + 8) * 2.0 ** -23 * abs(scale) * torch.einsum("hd,nhd->hn", qd.abs(), k.abs())).amax(1, keepdim=True)
        lse = torch.logsumexp(sc, 1)
        p = torch.exp(sc - lse[:, None])
        outs.append(torch.einsum("hn,nhd->hd", p, v))
        lses.append(lse)
        ws.append(p.reshape(cache.kvheads, G, n).sum(1))
        rel = 2 * es + 2.0 ** -20 + (n / 4 + 16) * 2.0 ** -23
        eo.append(rel * torch.einsum("hn,nhd->hd", p, v.abs()) + 1e-30)
        ew.append((p * rel).reshape(cache.kvheads, G, n).sum(1) + 1e-30)
    return outs, lses, ws, eo, ew


def evict64(weights, n, keep, recent):
    """Kept slots of one (sequence, KV head), ascending; NaN comes behind -inf."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    w = weights[:old].tolist()
    best = sorted(range(old), key=lambda i: (w[i] != w[i], 0 if w[i] != w[i] else -w[i], i))[: keep - recent]
    return sorted(best) + list(range(old, n))
