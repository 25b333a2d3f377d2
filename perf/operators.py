"""Operators of the paged key-value cache and of the logits, as they are measured.

Four operators of a serving step for several sequences, each at the sizes it meets:

  append      new key and value rows go to their slots in the cache's pages
  attention   new tokens attend to their sequence's cached positions; optionally every slot's
              accumulated attention weight grows by the weights the tokens gave it
  evict       a cache over its budget keeps its last slots and the slots of the largest weight
  logprobs    log probabilities of given tokens, the entropy and the likeliest alternatives

A cache layer is two pools of pages [pages][KV heads][slots][head_dim] (keys, values) and a table
[sequences][pages of a sequence] of page numbers.  `run` computes a case in plain torch operations,
or, where `own` is true, by this package's kernels.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = {"f32": 0, "f16": 1, "bf16": 30}  # GGML type numbers


def listed():
    def att(name, **kw):
        c = {"name": name, "op": "attention", "kind": "bf16", "seqs": 1, "heads": 32, "kvheads": 4, "head_dim": 128,
             "page": 16, "lo": 1, "hi": 1, "chunk": 1, "pad": 0, "weights": False}
        c.update(kw)
        return c

    return [
        # one chat stream a few hundred tokens in: latency counts
        att("attention 1x640 f16", kind="f16", lo=640, hi=640),
        # a serving step of 64 sequences at mixed depths of a 4096-token context
        att("attention 64x(130..4096) bf16", seqs=64, lo=130, hi=4096),
        # few sequences, long documents, larger pages
        att("attention 8x(9000..32768) bf16", seqs=8, page=64, lo=9000, hi=32768),
        # a 32-bit cache, three query heads to a KV head, a head size that is no power of two, an
        # empty sequence and rows of padding behind the last sequence
        att("attention 21x(0..1531) f32 d96", kind="f32", seqs=21, heads=12, kvheads=4, head_dim=96, page=24, lo=0,
            hi=1531, pad=3),
        # a serving step that keeps the slots' weights for a later eviction
        att("weights 32x(200..2500) f16", kind="f16", seqs=32, lo=200, hi=2500, weights=True),
        # the last 24 tokens of one long prompt, weights kept
        att("weights chunk 1x24x7001 bf16", lo=7001, hi=7001, chunk=24, page=32, weights=True),
        # a batch over its budget of 2048 slots, the last 256 kept in any case
        {"name": "evict 32x(1500..4096) bf16", "op": "evict", "kind": "bf16", "seqs": 32, "kvheads": 4, "head_dim": 128,
         "page": 16, "lo": 1500, "hi": 4096, "keep": 2048, "recent": 256},
        # one long sequence cut to an odd budget
        {"name": "evict 1x20011 f16", "op": "evict", "kind": "f16", "seqs": 1, "kvheads": 4, "head_dim": 128, "page": 32,
         "lo": 20011, "hi": 20011, "keep": 4999, "recent": 128},
        # a decode step's rows, and a prompt chunk of one sequence
        {"name": "append 64 bf16", "op": "append", "kind": "bf16", "seqs": 64, "kvheads": 4, "head_dim": 128, "page": 16,
         "rows": 1, "lo": 130, "hi": 4000},
        {"name": "append 3x1500 f16", "op": "append", "kind": "f16", "seqs": 3, "kvheads": 8, "head_dim": 128, "page": 16,
         "rows": 1500, "lo": 0, "hi": 700},
        # one sampled token with 20 alternatives over the 151,936-id vocabulary
        {"name": "logprobs 1x151936 top20", "op": "logprobs", "rows": 1, "vocab": 151936, "ids": 1, "top": 20, "scale": 2.5},
        # a pass of 128 rows, and of an odd vocabulary with several given tokens
        {"name": "logprobs 128x151936 top5", "op": "logprobs", "rows": 128, "vocab": 151936, "ids": 1, "top": 5,
         "scale": 2.5},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("attention", "attention", "weights", "evict", "append", "logprobs"))
    kind = rng.choice(("f32", "f16", "bf16"))
    if op == "logprobs":
        vocab = rng.choice((log(2, 1000), log(1000, 260000), 151936, 50257))
        rows = min(log(1, 512), max(1, 128 * 151936 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "ids": rng.randint(0, 4), "top": min(vocab, rng.randint(0, 64)),
                "scale": round(rng.uniform(0.3, 6.0), 2)}
    head_dim = rng.choice((32, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256))
    kvheads = rng.choice((1, 2, 3, 4, 4, 8))
    page = rng.choice((1, 5, 16, 16, 32, 64, 128, 250))
    size = {"f32": 4, "f16": 2, "bf16": 2}[kind]
    most = (1.5e8 if op == "evict" else 3e8) / (2 * kvheads * head_dim * size)  # slots of all sequences together
    seqs = log(1, 128)
    hi = max(1, min(log(1, 40000), int(most / seqs)))
    lo = rng.randint(0, hi)
    common = {"kind": kind, "seqs": seqs, "kvheads": kvheads, "head_dim": head_dim, "page": page}
    if op == "append":
        rows = max(1, min(log(1, 2000), hi, 6000 // seqs))
        return {"op": op, **common, "rows": rows, "lo": min(lo, hi - rows) if hi > rows else 0, "hi": max(0, hi - rows)}
    if op == "evict":
        keep = max(1, rng.randint(hi // 4, hi))
        return {"op": op, **common, "lo": lo, "hi": hi, "keep": keep, "recent": rng.randint(0, keep)}
    group = rng.choice((1, 2, 3, 4, 6, 8, 8, 12, 16))
    # (a prompt's last tokens: as many as the plain form has room for)
    most_rows = max(1, int(min(1e9 / (kvheads * hi * head_dim * 4), 1.5e10 / (4 * group * kvheads * hi * head_dim))))
    chunk = rng.choice((1, 1, 1, max(1, min(log(1, 32), hi, 256 // seqs, most_rows // seqs))))
    return {"op": "attention", **common, "heads": group * kvheads, "lo": max(lo, chunk if chunk > 1 else 0),
            "hi": max(hi, chunk), "chunk": chunk, "pad": rng.choice((0, 0, 3)), "weights": op == "weights"}


def lengths(case):
    """A length for each sequence, evenly from lo to hi."""
    n = case["seqs"]
    return [case["lo"] + (case["hi"] - case["lo"]) * i // max(1, n - 1) if n > 1 else case["hi"] for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * case["scale"]
        ids = torch.randint(0, vocab, (rows, case["ids"]), generator=g, device="cuda", dtype=torch.int32)
        return {"case": case, "logits": logits, "ids": ids,
                "logprobs": torch.zeros(rows, case["ids"], device="cuda"), "entropy": torch.zeros(rows, device="cuda"),
                "top_ids": torch.zeros(rows, case["top"], dtype=torch.int32, device="cuda"),
                "top_logprobs": torch.zeros(rows, case["top"], device="cuda")}
    S, KH, D, page, dt = case["seqs"], case["kvheads"], case["head_dim"], case["page"], DTYPES[case["kind"]]
    mix = torch.randperm(S, generator=g, device="cuda")
    lens = torch.tensor(lengths(case), dtype=torch.int32, device="cuda")[mix]
    most = case["hi"] + (case["rows"] if case["op"] == "append" else 0)
    max_pages = max(1, -(-most // page))
    dst_pages = -(-case["keep"] // page) if case["op"] == "evict" else 0
    n_pages = S * (max_pages + dst_pages) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    st = {"case": case, "lens": lens, "table": order[: S * max_pages].reshape(S, max_pages).contiguous(),
          "k": normal(n_pages, KH, page, D).to(dt), "v": normal(n_pages, KH, page, D).to(dt)}
    cap = max_pages * page
    if case["op"] == "append":
        n = S * case["rows"]
        st["seq"] = torch.arange(S, dtype=torch.int32, device="cuda").repeat_interleave(case["rows"])
        st["pos"] = (lens[:, None] + torch.arange(case["rows"], dtype=torch.int32, device="cuda")).reshape(-1).contiguous()
        st["new_k"], st["new_v"] = normal(n, KH, D), normal(n, KH, D)
        st["weights"] = normal(S, KH, cap).abs()
    elif case["op"] == "evict":
        # a few slots carry most of the weight, many carry nearly none, some exactly none
        w = torch.exp(2 * normal(S, KH, cap))
        st["weights"] = torch.where(torch.rand(S, KH, cap, generator=g, device="cuda") < 0.05, torch.zeros_like(w), w)
        wide = torch.full((S, max_pages), 0, dtype=torch.int32, device="cuda")
        n_dst = min(dst_pages, max_pages)
        wide[:, :n_dst] = order[S * max_pages: S * max_pages + S * dst_pages].reshape(S, dst_pages)[:, :n_dst]
        st["dst_table"] = wide
        st["weights_out"] = torch.zeros(S, KH, cap, device="cuda")
        st["kept"] = torch.zeros(S, KH, case["keep"], dtype=torch.int32, device="cuda")
        st["new_lens"] = torch.zeros(S, dtype=torch.int32, device="cuda")
    else:
        R, H, chunk = S * case["chunk"], case["heads"], case["chunk"]
        sharp = 0.5 + 2.0 * torch.rand(1, H, 1, generator=g, device="cuda")  # flat and peaked heads
        st["q"] = normal(R + case["pad"], H, D) * sharp
        none = torch.full((case["pad"],), -1, dtype=torch.int32, device="cuda")
        st["seq"] = torch.cat([torch.arange(S, dtype=torch.int32, device="cuda").repeat_interleave(chunk), none])
        back = torch.arange(chunk - 1, -1, -1, dtype=torch.int32, device="cuda")
        st["row_lens"] = torch.cat([(lens[:, None] - back).reshape(-1), none * 0]).contiguous()
        st["out"] = torch.zeros(R + case["pad"], H, D, device="cuda")
        st["lse"] = torch.zeros(R + case["pad"], H, device="cuda")
        if case["weights"]:
            st["weights"] = normal(S, KH, cap).abs()
    return st


def run(state):
    if own:
        return run_kernels(state)
    return {"append": plain_append, "evict": plain_evict, "attention": plain_attention, "logprobs": plain_logprobs}[
        state["case"]["op"]](state)


def dense(pool, table):
    """The pages of every sequence side by side: [sequences][KV heads][slots][head_dim]."""
    S, n = table.shape
    _, KH, page, D = pool.shape
    return pool[table.long()].transpose(1, 2).reshape(S, KH, n * page, D)


def plain_attention(st):
    c = st["case"]
    D, KH = c["head_dim"], c["kvheads"]
    G, cap = c["heads"] // KH, st["table"].shape[1] * c["page"]
    real = st["seq"] >= 0
    seq = st["seq"].clamp(min=0).long()
    k, v = dense(st["k"], st["table"]).float(), dense(st["v"], st["table"]).float()
    if c["chunk"] > 1 or c["pad"]:
        k, v = k[seq], v[seq]
    q = st["q"].reshape(-1, KH, G, D)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    seen = torch.arange(cap, device=s.device) < st["row_lens"][:, None, None, None]
    s = torch.where(seen, s, -torch.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    lse = (m + torch.log(total))[..., 0].reshape(-1, c["heads"])
    p = torch.where(total > 0, p / total, 0.0)
    out = torch.matmul(p, v).reshape(-1, c["heads"], D)
    out = torch.where(real[:, None, None], out, st["out"])
    lse = torch.where(real[:, None], torch.where(st["row_lens"][:, None] > 0, lse, -torch.inf), st["lse"])
    if not c["weights"]:
        return {"out": out, "lse": lse}
    given = torch.where(real[:, None, None], p.sum(2), 0.0)
    st["weights"].index_add_(0, seq, given)
    return {"out": out, "lse": lse, "weights": st["weights"]}


def plain_append(st):
    page = st["case"]["page"]
    seq, pos = st["seq"].long(), st["pos"].long()
    at, slot = st["table"][seq, pos // page].long(), pos % page
    st["k"][at, :, slot] = st["new_k"].to(st["k"].dtype)
    st["v"][at, :, slot] = st["new_v"].to(st["v"].dtype)
    st["weights"][seq, :, pos] = 0.0
    return {"k": st["k"], "v": st["v"], "weights": st["weights"]}


def plain_evict(st):
    c = st["case"]
    keep, page, w = c["keep"], c["page"], st["weights"]
    S, KH, cap = w.shape
    slot = torch.arange(cap, device=w.device)
    n = st["lens"][:, None, None]
    rank = torch.where(slot >= n, -torch.inf, torch.where(slot >= n - c["recent"], torch.inf, w))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(rank.gather(-1, order) > -torch.inf, order, cap).sort(-1).values
    if order.shape[-1] < keep:
        order = torch.cat([order, torch.full((S, KH, keep - order.shape[-1]), cap, device=w.device)], -1)
    some, order_in = order < cap, order.clamp(max=cap - 1)
    j = torch.arange(keep, device=w.device).clamp(max=cap - 1)
    at = st["dst_table"].long()[:, j // page]
    for pool in ("k", "v"):
        rows = dense(st[pool], st["table"]).gather(2, order_in[..., None].expand(-1, -1, -1, c["head_dim"]))
        old = st[pool][at[:, None], torch.arange(KH, device=w.device)[None, :, None], (j % page)[None, None]]
        few = min(keep, cap)
        new = torch.where(some[..., None], rows, old)[:, :, :few]
        st[pool][at[:, None, :few], torch.arange(KH, device=w.device)[None, :, None], (j % page)[None, None, :few]] = new
    few = min(keep, cap)
    st["weights_out"][..., :few] = torch.where(some, w.gather(-1, order_in), st["weights_out"][..., j])[..., :few]
    kept = torch.where(some, order, -1).to(torch.int32)
    return {"kept": kept, "new_lens": st["lens"].clamp(max=keep), "k": st["k"], "v": st["v"],
            "weights": st["weights_out"]}


def plain_logprobs(st):
    x = st["logits"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    log_total = torch.log(e.sum(-1, keepdim=True))
    lp = d - log_total
    entropy = -(torch.exp(lp) * lp).sum(-1)
    bits = (x + 0.0).view(torch.int32).long()  # (-0 counts as 0)
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    key = bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[-1], device=x.device))  # ties go to the lowest id
    top = torch.topk(key, st["case"]["top"], dim=-1).indices
    return {"logprobs": lp.gather(-1, st["ids"].long()), "entropy": entropy, "top_ids": top.to(torch.int32),
            "top_logprobs": lp.gather(-1, top)}


def run_kernels(st):
    from __graft_entry__ import load_package
    load_package()
    from qwen30brust_b200 import engine as E

    c, stream = st["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "logprobs":
        E.logprobs(st["logits"].data_ptr(), c["rows"], c["vocab"], ids_ptr=st["ids"].data_ptr(), n_ids=c["ids"],
                   top=c["top"], logprobs_ptr=st["logprobs"].data_ptr(), entropy_ptr=st["entropy"].data_ptr(),
                   top_ids_ptr=st["top_ids"].data_ptr(), top_logprobs_ptr=st["top_logprobs"].data_ptr(), stream=stream)
        return {"logprobs": st["logprobs"], "entropy": st["entropy"], "top_ids": st["top_ids"],
                "top_logprobs": st["top_logprobs"]}
    cache = E.PagedCache(KINDS[c["kind"]], st["k"].data_ptr(), st["v"].data_ptr(), st["k"].shape[0], c["page"],
                         c["kvheads"], c["head_dim"], st["table"].data_ptr(), c["seqs"], st["table"].shape[1])
    if c["op"] == "append":
        cache.append(st["new_k"].data_ptr(), st["new_v"].data_ptr(), st["pos"].numel(), st["pos"].data_ptr(),
                     seq_ptr=st["seq"].data_ptr(), weights_ptr=st["weights"].data_ptr(), stream=stream)
        return {"k": st["k"], "v": st["v"], "weights": st["weights"]}
    if c["op"] == "evict":
        cache.evict(st["weights"].data_ptr(), st["lens"].data_ptr(), c["keep"], c["recent"], st["kept"].data_ptr(),
                    st["new_lens"].data_ptr(), weights_out_ptr=st["weights_out"].data_ptr(),
                    dst_table_ptr=st["dst_table"].data_ptr(), stream=stream)
        return {"kept": st["kept"], "new_lens": st["new_lens"], "k": st["k"], "v": st["v"],
                "weights": st["weights_out"]}
    weights = st["weights"].data_ptr() if c["weights"] else None
    cache.attention(st["q"].data_ptr(), c["heads"], st["row_lens"].numel(), st["row_lens"].data_ptr(),
                    st["out"].data_ptr(), seq_ptr=st["seq"].data_ptr(), lse_ptr=st["lse"].data_ptr(),
                    weights_ptr=weights, stream=stream)
    out = {"out": st["out"], "lse": st["lse"]}
    return {**out, "weights": st["weights"]} if c["weights"] else out


def work(case):
    if case["op"] == "logprobs":
        rows, n = case["rows"], case["vocab"]
        return {"bytes": 4 * rows * (n + 2 * case["ids"] + 1 + 2 * case["top"]), "flops": 5 * rows * n}
    lens = lengths(case)
    row = case["kvheads"] * case["head_dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["kind"]]
    if case["op"] == "append":
        n = case["seqs"] * case["rows"]
        return {"bytes": n * (row * 2 * (4 + size) + 8 + 4 * case["kvheads"]), "flops": 0}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": kept * (row * 4 * size + 8 * case["kvheads"]) + 4 * case["kvheads"] * sum(lens), "flops": 0}
    chunk, H = case["chunk"], case["heads"]
    seen = sum(max(0, n - j) for n in lens for j in range(chunk))
    io = case["seqs"] * chunk * H * (2 * case["head_dim"] + 1) * 4
    weights = sum(lens) * case["kvheads"] * 8 if case["weights"] else 0
    return {"bytes": sum(lens) * row * 2 * size + io + weights, "flops": 4 * seen * H * case["head_dim"]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        return exact_logprobs(st)
    if case["op"] == "append":
        return exact_append(st)
    if case["op"] == "evict":
        return exact_evict(st)
    return exact_attention(st)


def exact_logprobs(st):
    rows = {"logprobs": [], "entropy": [], "top_logprobs": []}
    for x, ids in zip(st["logits"].double(), st["ids"].long()):
        lp = x - torch.logsumexp(x, 0)
        rows["logprobs"].append(lp[ids])
        rows["entropy"].append(-(lp.exp() * lp).sum())
        rows["top_logprobs"].append(lp.sort(descending=True).values[: st["case"]["top"]])
    return {k: torch.stack(v) for k, v in rows.items()}


def exact_append(st):
    k, v, w, page = st["k"].double(), st["v"].double(), st["weights"].double(), st["case"]["page"]
    table, at = st["table"].cpu(), 0
    for s, p in zip(st["seq"].tolist(), st["pos"].tolist()):
        g = int(table[s, p // page])
        k[g, :, p % page], v[g, :, p % page] = st["new_k"][at].to(st["k"].dtype).double(), st["new_v"][at].to(st["v"].dtype).double()
        w[s, :, p] = 0
        at += 1
    return {"k": k, "v": v, "weights": w}


def exact_evict(st):
    c = st["case"]
    keep, page = c["keep"], c["page"]
    kept = torch.full_like(st["kept"], -1)
    new_lens, out = st["new_lens"].clone(), st["weights_out"].double()
    pools = st["k"].clone(), st["v"].clone()
    for s, n in enumerate(st["lens"].tolist()):
        m = min(n, keep)
        new_lens[s] = m
        for h in range(c["kvheads"]):
            w = st["weights"][s, h, :n].double()
            if n <= keep:
                chosen = torch.arange(n, device=w.device)
            else:
                old = n - c["recent"]
                best = sorted(range(old), key=lambda i, w=w.tolist(): (-w[i], i))[: keep - c["recent"]]
                chosen = torch.tensor(sorted(best) + list(range(old, n)), device=w.device, dtype=torch.long)
            kept[s, h, :m] = chosen.to(torch.int32)
            out[s, h, :m] = w[chosen]
            to = torch.arange(m, device=w.device)
            a, b = st["table"][s].long()[chosen // page], st["dst_table"][s].long()[to // page]
            for old_pool, new_pool in zip((st["k"], st["v"]), pools):
                new_pool[b, h, to % page] = old_pool[a, h, chosen % page]
    return {"kept": kept, "new_lens": new_lens, "k": pools[0], "v": pools[1], "weights": out}


def exact_attention(st):
    c = st["case"]
    D, G, page = c["head_dim"], c["heads"] // c["kvheads"], c["page"]
    out, lse = st["out"].double(), st["lse"].double()
    weights = st["weights"].double() if c["weights"] else None
    n_of = st["row_lens"].tolist()
    for r, s in enumerate(st["seq"].tolist()):
        n = n_of[r]
        if s < 0:
            continue
        if n == 0:
            out[r], lse[r] = 0, -torch.inf
            continue
        at = torch.arange(n, device=out.device)
        g, slot = st["table"][s].long()[at // page], at % page
        k, v = st["k"][g, :, slot].double(), st["v"][g, :, slot].double()  # [n][KV heads][D]
        for h in range(c["heads"]):
            sc = (k[:, h // G] @ st["q"][r, h].double()) / math.sqrt(D)
            lse[r, h] = torch.logsumexp(sc, 0)
            p = torch.exp(sc - lse[r, h])
            out[r, h] = p @ v[:, h // G]
            if weights is not None:
                weights[s, h // G, :n] += p
    return {"out": out, "lse": lse, "weights": weights} if c["weights"] else {"out": out, "lse": lse}
