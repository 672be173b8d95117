"""CPU restatement, in 64 bits, of the paged-cache operators.

TEST INFRASTRUCTURE ONLY: imported by tests/ (as the checker of
fna2_b200/csrc/fna2_append.cu, fna2_paged.cu, fna2_keyweights.cu and
fna2_evict.cu); never by the product path.

The reference has no paged cache; this restates the op's definition
(FNA2/attention_fna2.py:94-170 for the norm and the rotation,
FNA2/flash_naylis_attn.py:99,159-165,192,195 for logits, GQA and normalisation)
for the last query rows of a sequence whose keys lie in pages.
"""
from __future__ import annotations

import math

import torch

EPS = 1e-6


def rows(pages, table, page_size, n):
    """The first n rows [n, heads, X] of one sequence, fp64."""
    j = torch.arange(n)
    return pages[table.long()[j // page_size], j % page_size].double()


def attention(x, causal, scale=None):
    """x: dict(kp, vp, rp, table, lens, cu, q, rq, gs) on the host.  Returns out [T, H, D],
    lse [H, T], key weights [B, H_KV, pages * page_size], all fp64."""
    q, kp = x["q"], x["kp"]
    T, H, D = q.shape
    page, h_kv = kp.shape[1], kp.shape[2]
    grp = H // h_kv
    hg = 0 if x["rp"] is None else x["rp"].shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((H, T), float("-inf"), dtype=torch.float64)
    w = torch.zeros(len(x["lens"]), h_kv, x["table"].shape[1] * page, dtype=torch.float64)
    cu = [int(c) for c in x["cu"]]
    for b, n_keys in enumerate(x["lens"]):
        n = cu[b + 1] - cu[b]
        k, v = (rows(x[p], x["table"][b], page, n_keys) for p in ("kp", "vp"))
        rk = rows(x["rp"], x["table"][b], page, n_keys) if hg else None
        i, j = torch.arange(n)[:, None], torch.arange(n_keys)[None]
        seen = (j <= n_keys - n + i) if causal else torch.ones(n, n_keys, dtype=torch.bool)
        for h in range(H):
            s = scale * q[cu[b]:cu[b + 1], h].double() @ k[:, h // grp].T
            if h < hg:
                s = s + float(x["gs"][h]) * (x["rq"][cu[b]:cu[b + 1], h].double() @ rk[:, h].T)
            for t in range(n):
                vis = seen[t]
                if not vis.any():
                    continue
                st = s[t][vis]
                m = st.max()
                e = torch.exp(st - m)
                l = e.sum() + EPS
                out[cu[b] + t, h] = (e / l) @ v[vis, h // grp]
                lse[h, cu[b] + t] = m + torch.log(l)
                w[b, h // grp, :n_keys][vis] += e / l
    return out, lse, w


def evict(weights, lens, budget, recent, sink):
    """Kept indices per sequence and KV head: lists of ascending slots."""
    kept = []
    for b, n in enumerate(lens):
        per_head = []
        for h in range(weights.shape[1]):
            old = max(0, n - recent)
            held = set(range(old, n)) | set(range(min(sink, old)))
            rest = [j for j in range(n) if j not in held]
            key = {j: float(weights[b, h, j]) for j in rest}
            rest.sort(key=lambda j: (key[j] != key[j], -key[j] if key[j] == key[j] else 0.0, j))
            per_head.append(sorted(list(held) + rest[:max(0, min(n, budget) - len(held))]))
        kept.append(per_head)
    return kept


def norm_rope(x, w, eps, inv_freq, pos):
    """x [T, heads, D] at positions pos [T], fp64 (w, inv_freq may be None)."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    if inv_freq is not None:
        ang = pos.double()[:, None, None] * torch.cat([inv_freq, inv_freq]).double()
        half = x.shape[-1] // 2
        x = x * torch.cos(ang) + torch.cat([-x[..., half:], x[..., :half]], -1) * torch.sin(ang)
    return x
