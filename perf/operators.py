"""Cases and plain forms of the paged-cache operators, for timing and comparison.

Four operators serve a model whose keys, values and relational factors R_k live in
pages of a pool:

  append   per-head RMSNorm and rotary embedding of new q and k rows, k / v / r_k
           written into the pages of their sequences
  attend   attention of each sequence's new tokens (one or thousands) over its pages,
           with the relational bias
  weights  attention weight each cached key received, summed over queries and the
           query heads of its KV head
  evict    per KV head, keep the keys of the largest accumulated weight (and the
           newest), compacted in order into fresh pages

``own`` selects the plain form (elementary torch operations in 32 bits) or the
framework's kernels.
"""
import math
import random

import torch

own = False

EPS = 1e-6       # O = acc / (l + EPS), LSE = m + log(l + EPS)
NORM_EPS = 1e-6  # RMSNorm
NEG = float("-inf")


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's new tokens of a batch of running sequences: 32 query heads on 8 KV heads
        dict(name="append decode", op="append", seqs=48, new=1, new_max=1, past=1000, page=64, H=32, HKV=8, HG=32,
             D=128, R=16, f32=False),
        # a packed prompt of several documents, fp32 activations, the model's default rank 32
        dict(name="append prompt", op="append", seqs=5, new=900, new_max=2500, past=0, page=128, H=16, HKV=16, HG=16,
             D=128, R=32, f32=True),
        # interactive use: one sequence, one token, a small model; latency is what counts
        dict(name="attend one", op="attend", seqs=1, new=1, new_max=1, past=257, past_min=257, page=16, H=4, HKV=4,
             HG=4, D=64, R=8, weights=False),
        # a decode step of a full batch with ragged lengths, gathering the weights that eviction needs
        dict(name="attend decode batch", op="attend", seqs=64, new=1, new_max=1, past=4096, past_min=64, page=64, H=32,
             HKV=8, HG=32, D=128, R=16, weights=True),
        # a single very long sequence decoded token by token, all heads separate
        dict(name="attend decode long", op="attend", seqs=1, new=1, new_max=1, past=131070, past_min=131070, page=128,
             H=32, HKV=32, HG=32, D=128, R=16, weights=False),
        # several drafted tokens of each sequence checked at once
        dict(name="attend verify", op="attend", seqs=16, new=3, new_max=7, past=2048, past_min=100, page=32, H=16,
             HKV=4, HG=12, D=128, R=16, weights=False),
        # one chunk of a long prompt over what is cached already, the model's default rank 32
        dict(name="attend prompt chunk", op="attend", seqs=1, new=2048, new_max=2048, past=30717, past_min=30717,
             page=128, H=32, HKV=32, HG=32, D=128, R=32, weights=False),
        # continuous batching: chunks of new prompts next to sequences that decode, a short and a long of each
        dict(name="attend mixed", op="attend", seqs=26, new=1, new_max=500, past=4000, past_min=1, page=64, H=16,
             HKV=16, HG=16, D=128, R=16, weights=False),
        # the last tokens of each prompt vote on which of its keys to keep
        dict(name="weights window", op="weights", seqs=4, new=64, new_max=64, past=16000, past_min=5000, page=64, H=32,
             HKV=8, HG=32, D=128, R=16),
        # every token of a prompt votes
        dict(name="weights prompt", op="weights", seqs=1, new=4095, new_max=4095, past=0, past_min=0, page=128, H=16,
             HKV=16, HG=16, D=128, R=32),
        # a few short sequences have outgrown their budget by some tokens
        dict(name="evict step", op="evict", seqs=4, past=600, past_min=450, budget=512, recent=64, sink=4, page=16, H=4,
             HKV=4, HG=4, D=64, R=8),
        # prompts cut to a fixed budget before decoding
        dict(name="evict prompt", op="evict", seqs=8, past=16384, past_min=8000, budget=4096, recent=256, sink=4,
             page=64, H=32, HKV=8, HG=32, D=128, R=16),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "weights", "evict"])
    hkv = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 1, 2, 4, 8])
    D = rng.choice([64, 128, 128])
    R = rng.choice([8, 16, 16, 24, 32])
    H = hkv * group if hkv * group <= 32 else hkv
    c = dict(op=op, page=rng.choice([16, 32, 64, 128]), H=H, HKV=hkv, HG=rng.choice([H, H, rng.randint(0, H)]), D=D,
             R=R)
    if op == "append":
        new = _log_int(rng, 1, 2000)
        c.update(seqs=_log_int(rng, 1, max(1, min(64, 8000 // new))), new=new, new_max=max(new, rng.randint(1, 2000)),
                 past=_log_int(rng, 1, 2000), f32=rng.random() < 0.5)
        c["new_max"] = min(c["new_max"], max(new, 8000 // c["seqs"]))
    elif op == "attend":
        new = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 2000)])
        past = _log_int(rng, 1, 30000)
        most = max(1, min(64, int(6e7 / ((past + new) * max(new, 16) * H / 16)), int(1e9 / ((past + new) * hkv * D))))
        c.update(new=new, new_max=new if rng.random() < 0.5 else new + rng.randint(0, new), past=past,
                 past_min=rng.randint(0, past), seqs=_log_int(rng, 1, most), weights=rng.random() < 0.3)
    elif op == "weights":
        new = _log_int(rng, 1, 1000)
        past = _log_int(rng, 1, 16000)
        most = max(1, min(16, int(6e7 / ((past + new) * max(new, 16) * H / 16)), int(1e9 / ((past + new) * hkv * D))))
        c.update(new=new, new_max=new, past=past, past_min=rng.randint(0, past), seqs=_log_int(rng, 1, most))
    else:
        past = _log_int(rng, 20, 16000)
        budget = max(4, int(past * rng.uniform(0.1, 1.1)))
        recent = rng.randint(0, budget // 2)
        c.update(past=past, past_min=rng.randint(0, past), budget=budget, recent=recent,
                 sink=rng.randint(0, min(8, budget - recent)),
                 seqs=_log_int(rng, 1, max(1, min(32, int(1.3e8 / (past * hkv * D))))))
    return c


def _lengths(case):
    """New tokens and tokens cached before them, per sequence (fixed by the case)."""
    rng = random.Random("%s %s %s" % (case["op"], case["seqs"], case["past"]))
    lo, hi = case.get("past_min", 0), case["past"]
    past = [rng.randint(lo, hi) for _ in range(case["seqs"])]
    past[0] = hi
    if case["op"] == "evict":
        return [0] * case["seqs"], past
    new = [rng.randint(case["new"], case["new_max"]) for _ in range(case["seqs"])]
    if case["op"] == "attend" and case["new"] == 1 and case["new_max"] > 64:  # mostly decoding sequences
        new = [n if i < 2 else 1 for i, n in enumerate(new)]
        new[0] = case["new_max"]
    return new, past


# --------------------------------------------------------------------------- inputs
class _Norm:  # what an RMSNorm module shows: its weight and eps
    def __init__(self, weight):
        self.weight, self.eps = weight, NORM_EPS


class _Rope:  # what a rotary embedding module shows: its frequencies
    def __init__(self, inv_freq):
        self.inv_freq = inv_freq


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    new, past = _lengths(case)
    op, page, H, HKV, HG, D, R = (case[k] for k in ("op", "page", "H", "HKV", "HG", "D", "R"))
    B, T = len(new), sum(new)
    bf = torch.bfloat16

    def randn(*shape, dtype=bf, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    total = [a + b for a, b in zip(new, past)]
    pages = [-(-n // page) for n in total]
    pages_out = -(-case["budget"] // page) * B if op == "evict" else 0
    order = torch.randperm(sum(pages) + pages_out + 3, device=dev, generator=g).to(torch.int32)  # pages lie anywhere
    table = torch.full((B, max(1, max(pages))), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    P = order.numel()
    s = dict(case=case, H=H, HKV=HKV, HG=HG, D=D, R=R, page=page, table=table,
             k_pages=randn(P, page, HKV, D), v_pages=randn(P, page, HKV, D),
             rk_pages=randn(P, page, HG, R, std=R ** -0.5) if HG else None,
             scale=1.0 / math.sqrt(D), max_new=max(new), max_len=max(total))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = ints(cu)
    s["lens_before"], s["lens"] = ints(past), ints(total)
    if op == "append":
        t = torch.float32 if case["f32"] else bf
        s.update(q=randn(T, H, D, dtype=t), k=randn(T, HKV, D, dtype=t), v=randn(T, HKV, D, dtype=t),
                 r_k=randn(T, HG, R, dtype=t, std=R ** -0.5) if HG else None,
                 q_norm=_Norm(1.0 + randn(D, dtype=torch.float32, std=0.2)),
                 k_norm=_Norm(1.0 + randn(D, dtype=torch.float32, std=0.2)),
                 rope=_Rope(10000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float32) / D)))
    elif op in ("attend", "weights"):
        s.update(q=randn(T, H, D), r_q=randn(T, HG, R, std=R ** -0.5) if HG else None,
                 gs=randn(HG, dtype=torch.float32) if HG else None, key_weights=None)
        if case.get("weights"):
            s["key_weights"] = torch.rand(B, HKV, table.shape[1] * page, device=dev, generator=g)
        if op == "weights":
            s["lse"] = _attend_plain(s)[1]  # of the attention that ran before
    else:
        w = torch.exp(randn(B, HKV, table.shape[1] * page, dtype=torch.float32, std=1.5))
        w[torch.rand(w.shape, device=dev, generator=g) < 0.03] = 0.0  # keys that nothing attended to
        s.update(key_weights=w, table_out=order[at:at + pages_out].reshape(B, -1).contiguous())
    if own:  # the handle of the page pool that a program makes once
        from fna2_b200.paged import PagedKV
        s["pool"] = PagedKV(s["k_pages"], s["v_pages"], s["rk_pages"])
    return s


def run(s):
    op = s["case"]["op"]
    return (_own if own else _plain)[op](s)


# --------------------------------------------------------------------------- the framework's calls
def _append_own(s):
    from fna2_b200.paged import qk_norm_rope_append
    q = qk_norm_rope_append(s["q"], s["k"], s["v"], s["pool"], s["table"], s["lens_before"], s["cu"], r_k=s["r_k"],
                            q_norm=s["q_norm"], k_norm=s["k_norm"], rope=s["rope"])
    return _append_out(s, q)


def _attend_own(s):
    from fna2_b200.paged import flash_naylis_paged
    out, lse = flash_naylis_paged(s["q"], s["pool"], s["table"], s["lens"], s["cu"], s["max_new"], r_q=s["r_q"],
                                  graph_scale=s["gs"], key_weights=s["key_weights"], return_lse=True,
                                  max_seqlen_k=s["max_len"])
    return (out, lse) if s["key_weights"] is None else (out, lse, s["key_weights"])


def _weights_own(s):
    from fna2_b200.paged import naylis_key_weights
    return naylis_key_weights(s["q"], s["lse"], s["pool"], s["table"], s["lens"], s["cu"], s["max_new"], r_q=s["r_q"],
                              graph_scale=s["gs"], max_seqlen_k=s["max_len"])


def _evict_own(s):
    from fna2_b200.paged import naylis_evict
    c = s["case"]
    kept, lens, w = naylis_evict(s["key_weights"], s["pool"], s["table"], s["lens"], c["budget"], s["table_out"],
                                 recent=c["recent"], sink=c["sink"], heads=s["H"], max_seqlen_k=s["max_len"])
    return _evict_out(s, kept, lens, w)


# --------------------------------------------------------------------------- plain forms
def _append_out(s, q):
    return [q, s["k_pages"], s["v_pages"]] + ([s["rk_pages"]] if s["HG"] else [])


def _evict_out(s, kept, lens, w):
    return [kept, lens, w, s["k_pages"], s["v_pages"]] + ([s["rk_pages"]] if s["HG"] else [])


def _token_seq(s):
    """Sequence of each packed token, and its index among that sequence's new tokens."""
    cu = s["cu"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, t - cu[b]


def _slots(s, b, j):
    """Page and slot in the page of key j of sequence b."""
    return s["table"].long()[b, j // s["page"]], j % s["page"]


def _append_plain(s):
    b, i = _token_seq(s)
    pos = s["lens_before"].long()[b] + i
    ang = pos.float()[:, None] * s["rope"].inv_freq
    cos, sin = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def norm_rope(x, norm):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + norm.eps) * norm.weight
        x1, x2 = x[..., :s["D"] // 2], x[..., s["D"] // 2:]
        return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).bfloat16()

    at = _slots(s, b, pos)
    s["k_pages"][at] = norm_rope(s["k"], s["k_norm"])
    s["v_pages"][at] = s["v"].bfloat16()
    if s["HG"]:
        s["rk_pages"][at] = s["r_k"].bfloat16()
    return _append_out(s, norm_rope(s["q"], s["q_norm"]))


def _gather(s, pages):
    """Rows of every sequence's pages, fp32, zero past its length: [B, L, heads, X]."""
    n = -(-s["max_len"] // s["page"])
    x = pages[s["table"][:, :n].long().clamp(min=0)].flatten(1, 2)[:, :s["max_len"]].float()
    dead = torch.arange(x.shape[1], device=x.device) >= s["lens"].long()[:, None]
    return x.masked_fill(dead[:, :, None, None], 0.0)


def _scores(s):
    """Masked logits [B, HKV, G, n, L] of the padded queries, and which padded rows are real."""
    cu, lens = s["cu"].long(), s["lens"].long()
    n_b = cu[1:] - cu[:-1]
    i = torch.arange(s["max_new"], device=cu.device)
    real = i < n_b[:, None]
    rows = torch.where(real, cu[:-1, None] + i, 0)
    B, H, HKV, HG = len(n_b), s["H"], s["HKV"], s["HG"]
    q = s["q"].float()[rows].unflatten(2, (HKV, H // HKV))
    S = torch.einsum("bnkgd,blkd->bkgnl", q, _gather(s, s["k_pages"])) * s["scale"]
    if HG:
        bias = torch.einsum("bnhr,blhr->bhnl", s["r_q"].float()[rows], _gather(s, s["rk_pages"]))
        S.view(B, H, *S.shape[3:])[:, :HG] += bias * s["gs"][:, None, None]
    seen = torch.arange(S.shape[-1], device=cu.device) <= (lens - n_b)[:, None, None] + i[None, :, None]
    return S.masked_fill_(~(seen & real[:, :, None])[:, None, None], NEG), real


def _attend_plain(s):
    S, real = _scores(s)
    m = S.amax(-1, keepdim=True)
    p = torch.exp(S - m.clamp(min=-1e30))
    l = p.sum(-1, keepdim=True) + EPS
    o = torch.einsum("bkgnl,blkd->bnkgd", p, _gather(s, s["v_pages"])) / l.movedim(3, 1)
    lse = torch.where(m > NEG, m + torch.log(l), NEG).squeeze(-1).flatten(1, 2)  # [B, H, n]
    out = o.flatten(2, 3)[real].bfloat16()
    lse_t = lse.movedim(2, 1)[real].t().contiguous()
    if s.get("key_weights") is not None and s["case"]["op"] == "attend":
        w = (p / l).sum((2, 3))
        s["key_weights"][:, :, :w.shape[-1]] += w
        return out, lse_t, s["key_weights"]
    return out, lse_t


def _weights_plain(s):
    S, real = _scores(s)
    cu = s["cu"].long()
    rows = torch.where(real, cu[:-1, None] + torch.arange(s["max_new"], device=cu.device), 0)
    lse = s["lse"].t()[rows].movedim(2, 1).unflatten(1, (s["HKV"], -1))[..., None]
    w = torch.exp(S - lse.clamp(min=-1e30)).sum((2, 3))
    full = torch.zeros(*w.shape[:2], s["table"].shape[1] * s["page"], device=w.device)
    full[:, :, :w.shape[-1]] = w
    return full


def _evict_plain(s):
    c, lens, L = s["case"], s["lens"].long(), s["max_len"]
    dev, B, HKV = lens.device, len(lens), s["HKV"]
    n_keep = lens.clamp(max=c["budget"])
    j = torch.arange(L, device=dev)
    w = s["key_weights"][:, :, :L]
    held = (j < c["sink"]) | (j >= (lens - c["recent"])[:, None])
    key = w.masked_fill(held[:, None], float("inf")).masked_fill((j >= lens[:, None])[:, None], NEG)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order).contiguous())
    kept = torch.where(rank < n_keep[:, None, None], j, L).sort(-1).values
    if L < c["budget"]:
        kept = torch.cat([kept, kept.new_full((B, HKV, c["budget"] - L), L)], -1)
    kept = kept[..., :c["budget"]]
    some = torch.arange(c["budget"], device=dev) < n_keep[:, None]
    b = torch.arange(B, device=dev)[:, None].expand_as(some)[some]
    dst = torch.arange(c["budget"], device=dev).expand_as(some)[some]
    to_page, to_slot = s["table_out"].long()[b, dst // s["page"]], dst % s["page"]
    src = kept.movedim(1, 2)[some]  # [rows, HKV]
    from_page, from_slot = s["table"].long()[b[:, None], src // s["page"]], src % s["page"]
    h = torch.arange(HKV, device=dev)
    for pages in (s["k_pages"], s["v_pages"]):
        pages[to_page, to_slot] = pages[from_page, from_slot, h]
    if s["HG"]:
        h = torch.arange(s["HG"], device=dev)
        of = h // (s["H"] // HKV)
        s["rk_pages"][to_page, to_slot] = s["rk_pages"][from_page[:, of], from_slot[:, of], h]
    w_out = torch.zeros(B, HKV, s["table_out"].shape[1] * s["page"], device=dev)
    w_out[:, :, :c["budget"]] = torch.where(some[:, None], w.gather(-1, kept.clamp(max=L - 1)), 0.0)
    return _evict_out(s, torch.where(some[:, None], kept, -1).int(), n_keep.int(), w_out)


_plain = dict(append=_append_plain, attend=_attend_plain, weights=_weights_plain, evict=_evict_plain)
_own = dict(append=_append_own, attend=_attend_own, weights=_weights_own, evict=_evict_own)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    new, past = _lengths(case)
    H, HKV, HG, D, R = (case[k] for k in ("H", "HKV", "HG", "D", "R"))
    T = sum(new)
    keys = sum(new) + sum(past)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    kv_row = 2 * 2 * HKV * D + 2 * HG * R
    if case["op"] == "append":
        e = 4 if case["f32"] else 2
        return dict(bytes=T * ((H + 2 * HKV) * D + HG * R) * (e + 2), flops=T * (H + HKV) * D * 8)
    if case["op"] == "attend":
        more = 8 * HKV * keys if case["weights"] else 0
        return dict(bytes=keys * kv_row + T * (4 * H * D + 2 * HG * R + 4 * H) + more,
                    flops=pairs * (4 * H * D + 2 * HG * R))
    if case["op"] == "weights":
        return dict(bytes=keys * (2 * HKV * D + 2 * HG * R + 4 * HKV) + T * (2 * H * D + 2 * HG * R + 4 * H),
                    flops=pairs * (2 * H * D + 2 * HG * R))
    kept = sum(min(p, case["budget"]) for p in past)
    return dict(bytes=keys * HKV * 4 + kept * (2 * kv_row + 8 * HKV), flops=keys * HKV)


# --------------------------------------------------------------------------- from the definitions, in 64 bits
def _rows64(s, b, pages, n):
    j = torch.arange(n, device=pages.device)
    return pages[s["table"][b].long()[j // s["page"]], j % s["page"]].double()


def _probabilities64(s, b, a, e):
    """Logits [H, n, len] of one sequence's queries in rows [a, e)."""
    n_keys, n = int(s["lens"][b]), e - a
    group = s["H"] // s["HKV"]
    k = _rows64(s, b, s["k_pages"], n_keys)
    S = s["q"][a:e].double().transpose(0, 1) @ k.repeat_interleave(group, 1).permute(1, 2, 0) / math.sqrt(s["D"])
    if s["HG"]:
        rk = _rows64(s, b, s["rk_pages"], n_keys)
        S[:s["HG"]] += s["gs"].double()[:, None, None] * (s["r_q"][a:e].double().transpose(0, 1) @ rk.permute(1, 2, 0))
    last = torch.arange(n_keys - n, n_keys, device=S.device)  # the last key that each query sees
    S[:, torch.arange(n_keys, device=S.device) > last[:, None]] = NEG
    return S


def exact(case, seed):
    s = prepare(case, seed)
    op, page, group = case["op"], s["page"], s["H"] // s["HKV"]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    if op == "evict":  # kept and lens are whole numbers; the rest are copies, without rounding
        names = [x for x in ("k_pages", "v_pages", "rk_pages") if s[x] is not None]
        pools = [s[x].double() for x in names]
        w_out = torch.zeros(len(lens), s["HKV"], s["table_out"].shape[1] * page, dtype=torch.float64, device="cuda")
        weights = s["key_weights"].tolist()
        for b, n in enumerate(lens):
            for h in range(s["HKV"]):
                w, n_old = weights[b][h], max(0, n - case["recent"])
                held = set(range(n_old, n)) | set(range(min(n, case["sink"])))
                ranked = sorted(set(range(n)) - held, key=lambda j: (-w[j], j))
                kept = sorted(sorted(held)[:case["budget"]] + ranked[:max(0, min(n, case["budget"]) - len(held))])
                w_out[b, h, :len(kept)] = torch.tensor([w[j] for j in kept], dtype=torch.float64, device="cuda")
                src, dst = torch.tensor(kept, dtype=torch.long, device="cuda"), torch.arange(len(kept), device="cuda")
                src = s["table"][b].long()[src // page], src % page
                dst = s["table_out"][b].long()[dst // page], dst % page
                for x, pool in zip(names, pools):
                    for y in ([h] if x != "rk_pages" else range(h * group, min(s["HG"], (h + 1) * group))):
                        pool[dst[0], dst[1], y] = s[x][src[0], src[1], y].double()
        return [None, None, w_out] + pools
    if op == "append":
        before = s["lens_before"].tolist()
        pools = [s[x].double() for x in ("k_pages", "v_pages", "rk_pages") if s[x] is not None]
        half = s["D"] // 2
        q_out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        for b, (a, e) in enumerate(zip(cu, cu[1:])):
            pos = torch.arange(before[b], before[b] + e - a, device=q_out.device)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=q_out.device),
                            pos.double()[:, None, None] * s["rope"].inv_freq.double())

            def turned(x, norm):
                x = x.double()
                x = x / (x.square().mean(-1, keepdim=True) + NORM_EPS).sqrt() * norm.weight.double()
                y = torch.complex(x[..., :half], x[..., half:]) * z
                return torch.cat([y.real, y.imag], -1)

            q_out[a:e] = turned(s["q"][a:e], s["q_norm"])
            at = s["table"][b].long()[pos // page], pos % page
            pools[0][at] = turned(s["k"][a:e], s["k_norm"])
            pools[1][at] = s["v"][a:e].double()
            if s["HG"]:
                pools[2][at] = s["r_k"][a:e].double()
        return [q_out] + pools
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(s["H"], cu[-1], dtype=torch.float64, device=out.device)
    w = torch.zeros(len(lens), s["HKV"], s["table"].shape[1] * page, dtype=torch.float64, device=out.device)
    for b, n_keys in enumerate(lens):
        v = _rows64(s, b, s["v_pages"], n_keys).repeat_interleave(group, 1).transpose(0, 1)
        for a in range(cu[b], cu[b + 1], 512):  # rows of the same sequence see keys up to their own place
            e = min(cu[b + 1], a + 512)
            own_lens = s["lens"]
            s["lens"] = own_lens - (cu[b + 1] - e)
            S = _probabilities64(s, b, a, e)
            s["lens"] = own_lens
            m = S.max(-1, keepdim=True).values
            l = torch.exp(S - m).sum(-1, keepdim=True) + EPS
            given = s["lse"][:, a:e, None].double() if op == "weights" else m + l.log()
            P = torch.exp(S - given)
            seen = S.shape[-1]
            w[b, :, :seen] += P.unflatten(0, (s["HKV"], group)).sum((1, 2))
            if op == "attend":
                out[a:e] = (P @ v[:, :seen]).transpose(0, 1)
                lse[:, a:e] = given.squeeze(-1)
    if op == "weights":
        return w
    if case["weights"]:
        return out, lse, s["key_weights"].double() + w
    return out, lse
