"""Serving one attention layer from a paged cache: prompts of several sequences go in by
chunks, the keys that nobody attends to are evicted, and decoding goes on with one token,
then with several drafted tokens at a time.

    python examples/paged_serving.py [--heads 16 --kv-heads 4 --chunk 512 --budget 1024]

The layer has random weights; what is printed is what a server would watch: cache lengths,
free pages and the time per step.  Before anything is evicted, the chunked prompt is
compared with the packed prefill op over whole prompts.
"""
import argparse
import os
import sys
import time

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fna2_b200 import flash_naylis_attn  # noqa: E402
from fna2_b200.paged import NaylisPagedCache  # noqa: E402
from fna2_b200.qk_prep import apply_qk_norm_rope_varlen  # noqa: E402
from fna2_b200.rel_proj import compute_rq_rk  # noqa: E402


class Norm(nn.Module):
    def __init__(self, dim):
        super().__init__()
        self.weight, self.eps = nn.Parameter(torch.ones(dim)), 1e-6


class Rope(nn.Module):
    def __init__(self, dim):
        super().__init__()
        self.register_buffer("inv_freq", 10000.0 ** (-torch.arange(0, dim, 2).float() / dim))


class Layer(nn.Module):
    """The projections of a Naylis attention layer (no bias terms)."""

    def __init__(self, embed, heads, kv_heads, head_dim, rank):
        super().__init__()
        self.h, self.kv, self.d, self.r = heads, kv_heads, head_dim, rank
        self.qkv = nn.Linear(embed, (heads + 2 * kv_heads) * head_dim, bias=False)
        self.rel = nn.Parameter(torch.randn(2 * heads * rank, embed) * 0.05)
        self.graph_scale = nn.Parameter(torch.randn(heads))
        self.q_norm, self.k_norm, self.rope = Norm(head_dim), Norm(head_dim), Rope(head_dim)
        self.out = nn.Linear(heads * head_dim, embed, bias=False)

    def project(self, x):
        q, k, v = self.qkv(x).unflatten(-1, (-1, self.d)).split([self.h, self.kv, self.kv], dim=-2)
        r_q, r_k = compute_rq_rk(x, self.rel.to(x.dtype), self.h, self.r)
        return q, k, v, r_q, r_k

    def serve(self, x, new, cache):
        """new[b] tokens of each sequence, packed in x."""
        q, k, v, r_q, r_k = self.project(x)
        q = cache.append(q, k, v, new, r_k, self.q_norm, self.k_norm, self.rope)
        return self.out(cache.attend(q, r_q, self.graph_scale.float()).flatten(1))

    def prefill(self, x, lengths):
        """The same over whole prompts, with the packed ops."""
        q, k, v, r_q, r_k = self.project(x)
        cu = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32, device=x.device)
        q, k = apply_qk_norm_rope_varlen(q, k, cu, self.q_norm, self.k_norm, self.rope)
        o = flash_naylis_attn(q, k, v, r_q, r_k, self.graph_scale.float(), is_causal=True, cu_seqlens_q=cu,
                              cu_seqlens_k=cu, max_seqlen_q=max(lengths), max_seqlen_k=max(lengths))
        return self.out(o.flatten(1))


@torch.no_grad()
def run(heads=16, kv_heads=4, head_dim=128, rank=16, embed=1024, prompts=(1900, 300, 1024, 77), chunk=512, budget=1024,
        recent=64, sink=4, steps=32, drafted=4, seed=0, verbose=True):
    """Returns what the run measured: the chunked prompt's largest deviation from the packed
    prefill (relative to the largest output) and the final cache lengths."""
    torch.manual_seed(seed)
    layer = Layer(embed, heads, kv_heads, head_dim, rank).cuda().bfloat16()
    for m in (layer.q_norm, layer.k_norm, layer.rope):
        m.float()
    B, page = len(prompts), 64
    most = max(prompts) + steps * (1 + drafted)
    cache = NaylisPagedCache(2 * B * (-(-most // page)), page, B, most, heads, kv_heads, head_dim, heads, rank)
    x = [torch.randn(n, embed, device="cuda").bfloat16() for n in prompts]

    def say(*a):
        if verbose:
            print(*a, flush=True)

    done, outs = [0] * B, [[] for _ in range(B)]
    while any(d < n for d, n in zip(done, prompts)):  # sequences of any progress share a call
        new = [min(chunk, n - d) for d, n in zip(done, prompts)]
        o = layer.serve(torch.cat([s[d:d + n] for s, d, n in zip(x, done, new)]), new, cache)
        for b, piece in enumerate(o.split(new)):
            outs[b].append(piece)
        done = [d + n for d, n in zip(done, new)]
    chunked, whole = torch.cat([torch.cat(p) for p in outs]).float(), layer.prefill(torch.cat(x), prompts).float()
    off = ((chunked - whole).abs().max() / whole.abs().max()).item()
    say(f"prompts {list(prompts)} in chunks of {chunk}: largest deviation from the packed prefill {off:.2e}")
    cut = cache.evict(budget, recent, sink)
    say(f"evicted to {budget}: slots {cut}, lengths {cache.lengths}, {cache.free_pages} pages free")

    last = torch.stack([s[-1] for s in x])
    for n in (1, drafted):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(steps):
            o = layer.serve(last.repeat_interleave(n, 0), [n] * B, cache)
            last = torch.nn.functional.normalize(o.view(B, n, embed)[:, -1].float(), dim=-1).mul(embed ** 0.5).bfloat16()
        torch.cuda.synchronize()
        say(f"{steps} steps of {n} token(s) per sequence: {(time.perf_counter() - t) / steps * 1e6:.0f} us each, "
            f"lengths {cache.lengths}")
    cache.evict(budget, recent, sink)
    assert torch.isfinite(last).all()
    return dict(deviation=off, lengths=list(cache.lengths), device_lengths=cache.seqlens.tolist(),
                positions=cache.positions.tolist(), free_pages=cache.free_pages)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("heads", 16), ("kv-heads", 4), ("head-dim", 128), ("rank", 16), ("embed", 1024), ("chunk", 512),
                          ("budget", 1024), ("recent", 64), ("sink", 4), ("steps", 32), ("drafted", 4), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=default)
    run(**vars(ap.parse_args()))
