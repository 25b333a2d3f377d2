"""The model's forward in 64 bits (model.rs:217-302) with a cache that can be held to a budget: every layer and KV
head has slots of its own, each with its key, value and accumulated attention weight."""
import numpy as np

from golden.make_golden import dequantize_all


class Bounded:
    """One sequence.  wrong: a mistake to make on purpose, to see that it shows."""

    def __init__(self, img, spec, oracle, wrong=""):
        self.w = {k: v.astype(np.float64) for k, v in dequantize_all(img, oracle).items()}
        self.s, self.wrong, self.position = spec, wrong, 0
        self.slots = [[{"k": [], "v": [], "w": []} for _ in range(spec.kvheads)] for _ in range(spec.layers)]
        self.margin = np.inf  # the smallest distance of a choice (experts, slots) from another one

    def rms(self, x, w):
        return x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + self.s.eps) * w

    def rope(self, x):
        half = self.s.head_dim // 2
        angle = self.position * self.s.theta ** (-2.0 * np.arange(half) / self.s.head_dim)
        a, b = x[:, :half], x[:, half:]
        return np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], 1)

    def forward(self, token):
        s, w = self.s, self.w
        x = w["token_embd.weight"][token].copy()
        for i in range(s.layers):
            p = f"blk.{i}."
            xn = self.rms(x, w[p + "attn_norm.weight"])
            q = (w[p + "attn_q.weight"] @ xn).reshape(s.heads, s.head_dim)
            k = (w[p + "attn_k.weight"] @ xn).reshape(s.kvheads, s.head_dim)
            v = (w[p + "attn_v.weight"] @ xn).reshape(s.kvheads, s.head_dim)
            q = self.rope(self.rms(q, w[p + "attn_q_norm.weight"]))
            k = self.rope(self.rms(k, w[p + "attn_k_norm.weight"]))
            out = np.empty_like(q)
            group = s.heads // s.kvheads
            for h, c in enumerate(self.slots[i]):
                c["k"].append(k[h]), c["v"].append(v[h]), c["w"].append(0.0)
                sc = q[h * group:(h + 1) * group] @ np.stack(c["k"]).T / np.sqrt(s.head_dim)
                pr = np.exp(sc - sc.max(1, keepdims=True))
                pr /= pr.sum(1, keepdims=True)
                out[h * group:(h + 1) * group] = pr @ np.stack(c["v"])
                c["w"] = (np.array(c["w"]) + pr.sum(0)).tolist()
            x = x + w[p + "attn_output.weight"] @ out.reshape(-1)
            xn = self.rms(x, w[p + "ffn_norm.weight"])
            r = w[p + "ffn_gate_inp.weight"] @ xn
            order = np.argsort(-r, kind="stable")
            ids = order[:s.top]
            self.margin = min(self.margin, r[order[s.top - 1]] - r[order[s.top]])
            pw = np.exp(r[ids] - r[ids].max())
            pw /= pw.sum()
            for e, g in zip(ids, pw):
                a = w[p + "ffn_gate_exps.weight"][e] @ xn
                x = x + g * (w[p + "ffn_down_exps.weight"][e] @ (a / (1 + np.exp(-a)) * (w[p + "ffn_up_exps.weight"][e] @ xn)))
        self.position += 1
        out = w["output.weight"] if "output.weight" in w else w["token_embd.weight"]
        return out @ self.rms(x, w["output_norm.weight"])

    def evict(self, keep, recent):
        chosen = {}
        for i, layer in enumerate(self.slots):
            for h, c in enumerate(layer):
                n = len(c["w"])
                if n <= keep:
                    continue
                last = 0 if self.wrong == "no recent" else recent
                weights = np.array((self.slots[0][h] if self.wrong == "layer 0" else c)["w"][:n - last])
                order = np.argsort(weights if self.wrong == "smallest" else -weights, kind="stable")
                if 0 < keep - last < n - last:
                    a, b = weights[order[keep - last - 1]], weights[order[keep - last]]
                    self.margin = min(self.margin, abs(a - b) / max(a, b))
                kept = sorted(order[:keep - last].tolist()) + list(range(n - last, n))
                if self.wrong == "one head's slots":
                    kept = chosen.setdefault(i, kept)
                chosen[i, h] = kept
        for (i, h), kept in [x for x in chosen.items() if isinstance(x[0], tuple)]:
            c = self.slots[i][h]
            for f in ("k", "v"):
                c[f] = [c[f][j] for j in kept]
            c["w"] = c["w"][:keep] if self.wrong == "weights stay" else [c["w"][j] for j in kept]
