"""Serving from a paged cache of K, V and R_k, with the relational bias.

The reference has no such path: its decode step (FNA2/attention_fna2.py:428-432)
grows a contiguous cache by concatenation, drops graph_bias and takes one token.
Here the caches of many sequences lie in pages of one pool, and four operators
work on them, each one call into libfna2_b200.so:

    qk_norm_rope_append   QK-RMSNorm + RoPE of new tokens at their positions, and
                          their k, v, r_k written into the pages
    flash_naylis_paged    attention of the new tokens (one or thousands per sequence)
                          over the pages
    naylis_key_weights    attention weight that each cached key received
    naylis_evict          keep the keys of the largest weight and the newest

Key j of sequence b is slot j % page_size of page page_table[b, j // page_size].
New token i of the n that sequence b adds sees key j iff j <= len - n + i, where
len = cache_seqlens[b] counts the new tokens: the rows equal the last n rows of
flash_naylis_attn over the whole sequence.  Sequence lengths and page tables are
int32 on the device and are never read on the host; a sequence whose lengths
break the bounds of a call is skipped and a status recorded (fna2_device_status:
631 append, 641 attention and key weights, 651 eviction).

NaylisPagedCache keeps the pool, the tables and the lengths, and runs the four.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib

_DT = {torch.float32: _lib.FNA2_DTYPE_F32, torch.bfloat16: _lib.FNA2_DTYPE_BF16}


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _want(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _rows_ok(t: torch.Tensor, name: str, heads: int, cols: int, tokens: Optional[int] = None) -> None:
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != cols or (tokens is not None and t.shape[0] != tokens):
        raise ValueError(f"{name} must be [{'T' if tokens is None else tokens}, {heads}, {cols}] "
                         f"(got {tuple(t.shape)})")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Unit column stride, 16-byte aligned rows; anything else is copied once."""
    vec = 16 // t.element_size()
    s = t.stride()
    if s[2] != 1 or s[0] % vec or s[1] % vec or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _int32(t: torch.Tensor, name: str, n: int) -> torch.Tensor:
    if t.dtype != torch.int32 or not t.is_cuda or t.numel() != n:
        raise ValueError(f"{name} must be a CUDA int32 tensor of {n} entries")
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, name: str = "page_table") -> torch.Tensor:
    if t.dtype != torch.int32 or not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name} must be a CUDA int32 tensor [batch, pages]")
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class PagedKV:
    """A pool of pages: k_pages, v_pages [P, page_size, H_KV, D] and, with graph heads,
    rk_pages [P, page_size, H_G, R], bf16, unit column stride, other strides multiples
    of 8 (a pool kept as [P, H_KV, page_size, D] is passed as .transpose(1, 2)).
    page_size: a power of two, 16 to 1024.  The handle checks the tensors once."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, rk_pages: Optional[torch.Tensor] = None):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("rk_pages", rk_pages)):
            if t is None:
                continue
            if t.dtype != torch.bfloat16:
                raise TypeError(f"{name} must be bfloat16 (got {t.dtype})")
            _want(t.is_cuda, f"{name} must be a CUDA tensor")
            _want(t.dim() == 4, f"{name} must be [pages, page_size, heads, columns] (got {tuple(t.shape)})")
            _want(t.stride(3) == 1, f"{name} must have unit stride in its last dim")
            _want(t.shape[:2] == k_pages.shape[:2], f"{name} must have the pages and page size of k_pages")
        _want(v_pages.shape == k_pages.shape, "v_pages must have the shape of k_pages")
        self.k_pages, self.v_pages, self.rk_pages = k_pages, v_pages, rk_pages
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = k_pages.shape
        self.graph_heads, self.rank = (0, 16) if rk_pages is None else rk_pages.shape[2:]
        if self.graph_heads == 0:
            rk_pages = None
        self.device = k_pages.device
        c = _lib.Fna2PagedKV(self.num_pages, self.page_size, self.kv_heads, self.graph_heads, self.head_dim, self.rank)
        c.k, c.v, c.rk = k_pages.data_ptr(), v_pages.data_ptr(), _ptr(rk_pages)
        c.k_page_stride, c.k_token_stride, c.k_head_stride = k_pages.stride()[:3]
        c.v_page_stride, c.v_token_stride, c.v_head_stride = v_pages.stride()[:3]
        if rk_pages is not None:
            c.rk_page_stride, c.rk_token_stride, c.rk_head_stride = rk_pages.stride()[:3]
        self._c = c
        self._ref = ctypes.byref(c)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pool: PagedKV, page_table: torch.Tensor,
                        cache_seqlens: torch.Tensor, cu_seqlens: torch.Tensor, r_k: Optional[torch.Tensor] = None,
                        positions: Optional[torch.Tensor] = None, q_norm=None, k_norm=None, rope=None) -> torch.Tensor:
    """New tokens into the cache.

    q [T, H, D], k, v [T, H_KV, D], r_k [T, H_G, R] (fp32 or bf16, one dtype), packed by
    cu_seqlens [B+1].  q and k go through the norms and the rotary embedding exactly as in
    apply_qk_norm_rope_varlen (``q_norm``/``k_norm``: modules with .weight and .eps, or None;
    ``rope``: a module with .inv_freq, or None), at position positions[b] + i (None:
    cache_seqlens[b] + i) for new token i; then k, v, r_k are written as bf16 into slots
    cache_seqlens[b] + i (slots in use before the call; the caller advances it).
    Returns q as bf16 [T, H, D].  Rows of tokens outside [cu[0], cu[B]) are not written."""
    _want(q.dtype in _DT and k.dtype == q.dtype and v.dtype == q.dtype and (r_k is None or r_k.dtype == q.dtype),
          "q, k, v, r_k: fp32 or bf16, same dtype")
    T, H, D = q.shape if q.dim() == 3 else (0, 0, 0)
    _rows_ok(q, "q", H, pool.head_dim)
    _rows_ok(k, "k", pool.kv_heads, pool.head_dim, T)
    _rows_ok(v, "v", pool.kv_heads, pool.head_dim, T)
    _want((r_k is not None) == (pool.graph_heads > 0), "r_k goes with a pool that has rk_pages")
    if r_k is not None:
        _rows_ok(r_k, "r_k", pool.graph_heads, pool.rank, T)
        r_k = _aligned(r_k)
    _want((q_norm is None) == (k_norm is None), "give both norms or neither")
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    table = _table(page_table)
    B = table.shape[0]
    lens, cu = _int32(cache_seqlens, "cache_seqlens", B), _int32(cu_seqlens, "cu_seqlens", B + 1)
    out = torch.empty((T, H, D), dtype=torch.bfloat16, device=q.device)
    a = _lib.Fna2AppendArgs(B, H, table.shape[1], _DT[q.dtype], _lib.FNA2_DTYPE_F32, _DT[q.dtype], T)
    a.q = _lib.Fna2Rows(q.data_ptr(), q.stride(0), q.stride(1))
    a.k = _lib.Fna2Rows(k.data_ptr(), k.stride(0), k.stride(1))
    a.v = _lib.Fna2Rows(v.data_ptr(), v.stride(0), v.stride(1))
    if r_k is not None:
        a.r_k = _lib.Fna2Rows(r_k.data_ptr(), r_k.stride(0), r_k.stride(1))
    a.q_out = _lib.Fna2Rows(out.data_ptr(), H * D, D)
    a.page_table, a.table_stride = table.data_ptr(), table.stride(0)
    a.cache_seqlens, a.cu_seqlens = lens.data_ptr(), cu.data_ptr()
    if positions is not None:
        positions = _int32(positions, "positions", B)
        a.positions = positions.data_ptr()
    if q_norm is not None:
        wq, wk = q_norm.weight.detach(), k_norm.weight.detach()
        _want(wq.dtype in _DT and wk.dtype == wq.dtype and wq.numel() == D and wk.numel() == D,
              "norm weights: fp32 or bf16 [head_dim], same dtype")
        _want(float(q_norm.eps) == float(k_norm.eps), "the two norms must share eps")
        wq, wk = wq.contiguous(), wk.contiguous()
        a.weight_dtype, a.rope_dtype = _DT[wq.dtype], _DT[torch.promote_types(q.dtype, wq.dtype)]
        a.q_weight, a.k_weight, a.eps = wq.data_ptr(), wk.data_ptr(), float(q_norm.eps)
    if rope is not None:
        f = rope.inv_freq.detach()
        if f.dtype != torch.float32 or f.device != q.device or not f.is_contiguous():
            f = f.to(device=q.device, dtype=torch.float32).contiguous()
        _want(f.numel() == D // 2, "rope.inv_freq must have head_dim / 2 entries")
        a.inv_freq = f.data_ptr()
    rc = _lib.load().fna2_paged_append(pool._ref, ctypes.byref(a), _stream(q.device))
    if rc:
        _lib.check(rc, "fna2_paged_append")
    return out


def _attn_args(q, pool, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, r_q, graph_scale, softmax_scale,
               is_causal, key_weights, max_seqlen_k):
    """The argument block of an attention or key weights call, and the tensors it points into."""
    if q.dtype != torch.bfloat16 or (r_q is not None and r_q.dtype != torch.bfloat16):
        raise TypeError("q and r_q must be bfloat16")
    T, H, D = q.shape if q.dim() == 3 else (0, 0, 0)
    _rows_ok(q, "q", H, pool.head_dim)
    q = _aligned(q)
    table = _table(page_table)
    B, max_pages = table.shape
    lens, cu = _int32(cache_seqlens, "cache_seqlens", B), _int32(cu_seqlens_q, "cu_seqlens_q", B + 1)
    capacity = max_pages * pool.page_size
    max_k = capacity if max_seqlen_k is None else min(int(max_seqlen_k), capacity)
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    a = _lib.Fna2PagedAttnArgs(B, H, T, int(max_seqlen_q), max_k, max_pages, 1 if is_causal else 0, 0, scale,
                               table.data_ptr(), table.stride(0), lens.data_ptr(), cu.data_ptr(),
                               q.data_ptr(), q.stride(0), q.stride(1))
    gs = None
    if pool.graph_heads:
        _want(r_q is not None and graph_scale is not None, "graph heads need r_q and graph_scale")
        _rows_ok(r_q, "r_q", pool.graph_heads, pool.rank, T)
        r_q = _aligned(r_q)
        gs = graph_scale.detach()
        _want(gs.numel() == pool.graph_heads and gs.is_cuda, "graph_scale must be a CUDA tensor [H_G]")
        if gs.dtype != torch.float32 or not gs.is_contiguous():
            gs = gs.float().contiguous()
        a.r_q, a.rq_token_stride, a.rq_head_stride = r_q.data_ptr(), r_q.stride(0), r_q.stride(1)
        a.graph_scale = gs.data_ptr()
    else:
        _want(r_q is None, "r_q goes with a pool that has rk_pages")
    if key_weights is not None:
        if key_weights.dtype != torch.float32 or not key_weights.is_cuda or key_weights.dim() != 3 or \
                key_weights.shape[:2] != (B, pool.kv_heads) or key_weights.shape[2] < max_k or \
                key_weights.stride(2) != 1:
            raise ValueError(f"key_weights must be CUDA fp32 [{B}, {pool.kv_heads}, >= {max_k}] with unit stride "
                             "in its last dim")
        a.key_weights = key_weights.data_ptr()
        a.kw_batch_stride, a.kw_head_stride = key_weights.stride(0), key_weights.stride(1)
    return a, (q, r_q, gs, table, lens, cu)


def _workspace(size_fn, pool, a, device):
    n = size_fn(pool._ref, ctypes.byref(a))
    if n == 0:
        if _lib.load().fna2_last_error():
            raise RuntimeError(_lib.load().fna2_last_error().decode())
        return None, 0
    return torch.empty(n, dtype=torch.uint8, device=device), n


def flash_naylis_paged(q: torch.Tensor, pool: PagedKV, page_table: torch.Tensor, cache_seqlens: torch.Tensor,
                       cu_seqlens_q: torch.Tensor, max_seqlen_q: int, r_q: Optional[torch.Tensor] = None,
                       graph_scale: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                       is_causal: bool = True, key_weights: Optional[torch.Tensor] = None, return_lse: bool = False,
                       max_seqlen_k: Optional[int] = None, num_splits: int = 0):
    """Attention of new tokens over a paged cache.

    q [T, H, D], r_q [T, H_G, R] bf16, packed by cu_seqlens_q [B+1]; cache_seqlens [B] counts
    the new tokens, whose keys are already in the pages.  max_seqlen_q bounds the new tokens of
    a sequence, max_seqlen_k (None: what a page table row holds) its cached keys.  Causal: new
    token i of n sees keys j <= len - n + i; otherwise every key (e.g. an encoder's states).  A
    row that sees no key gets out 0, lse -inf.  key_weights (fp32 [B, H_KV, >= max_seqlen_k]):
    the attention weight that each key received, summed over the new tokens and the query
    heads of its KV head, is added to it.
    Returns out [T, H, D] bf16 (and lse fp32 [H, T] if return_lse)."""
    a, held = _attn_args(q, pool, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, r_q, graph_scale,
                         softmax_scale, is_causal, key_weights, max_seqlen_k)
    T, H, D = q.shape
    a.num_splits = num_splits
    out = torch.empty((T, H, D), dtype=torch.bfloat16, device=q.device)
    a.out, a.out_token_stride, a.out_head_stride = out.data_ptr(), H * D, D
    lse = None
    if return_lse:
        lse = torch.empty((H, T), dtype=torch.float32, device=q.device)
        a.lse, a.lse_head_stride = lse.data_ptr(), T
    lib = _lib.load()
    ws, n = _workspace(lib.fna2_paged_attn_workspace_size, pool, a, q.device)
    rc = lib.fna2_paged_attn(pool._ref, ctypes.byref(a), _ptr(ws), n, _stream(q.device))
    if rc:
        _lib.check(rc, "fna2_paged_attn")
    return (out, lse) if return_lse else out


def naylis_key_weights(q: torch.Tensor, lse: torch.Tensor, pool: PagedKV, page_table: torch.Tensor,
                       cache_seqlens: torch.Tensor, cu_seqlens_q: torch.Tensor, max_seqlen_q: int,
                       r_q: Optional[torch.Tensor] = None, graph_scale: Optional[torch.Tensor] = None,
                       softmax_scale: Optional[float] = None, is_causal: bool = True,
                       key_weights: Optional[torch.Tensor] = None, max_seqlen_k: Optional[int] = None) -> torch.Tensor:
    """Attention weight that each cached key received from the given queries.

    Arguments as in flash_naylis_paged; lse [H, T] fp32 is the LSE of those queries over the
    same keys.  The queries may be the last tokens of each sequence only (they vote for the
    rest).  Adds to key_weights, or to zeros [B, H_KV, pages * page_size] when None; returns it."""
    if key_weights is None:
        key_weights = torch.zeros((page_table.shape[0], pool.kv_heads, page_table.shape[1] * pool.page_size),
                                  dtype=torch.float32, device=q.device)
    a, held = _attn_args(q, pool, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, r_q, graph_scale,
                         softmax_scale, is_causal, key_weights, max_seqlen_k)
    if lse.dtype != torch.float32 or not lse.is_cuda or tuple(lse.shape) != (q.shape[1], q.shape[0]):
        raise ValueError(f"lse must be CUDA fp32 [{q.shape[1]}, {q.shape[0]}] (got {lse.dtype} {tuple(lse.shape)})")
    if lse.stride(1) != 1:
        lse = lse.contiguous()
    a.lse, a.lse_head_stride = lse.data_ptr(), lse.stride(0)
    lib = _lib.load()
    ws, n = _workspace(lib.fna2_key_weights_workspace_size, pool, a, q.device)
    rc = lib.fna2_key_weights(pool._ref, ctypes.byref(a), _ptr(ws), n, _stream(q.device))
    if rc:
        _lib.check(rc, "fna2_key_weights")
    return key_weights


def naylis_evict(key_weights: torch.Tensor, pool: PagedKV, page_table: torch.Tensor, cache_seqlens: torch.Tensor,
                 budget: int, page_table_out: torch.Tensor, recent: int = 0, sink: int = 0,
                 heads: Optional[int] = None,
                 max_seqlen_k: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keep, per sequence and KV head, min(len, budget) keys: the first `sink`, the last
    `recent`, and of the others those of the largest key_weights [B, H_KV, >= max_seqlen_k]
    (ties to the lowest index, NaN below every number).  Their rows of K, V and R_k are copied
    in order to slots [0, kept) of the pages of page_table_out [B, >= budget / page_size], which
    must be pages that no sequence of the call occupies; the old pages are the caller's to
    free.  heads: query heads (None: graph heads, or KV heads if there are none), which fixes
    whose R_k moves with a KV head.
    Returns kept [B, H_KV, budget] int32 (-1 past the count), the new lengths [B] int32, and the
    kept keys' weights [B, H_KV, pages_out * page_size] (0 past the count)."""
    table, table_out = _table(page_table), _table(page_table_out, "page_table_out")
    B, max_pages = table.shape
    _want(table_out.shape[0] == B, "page_table_out must have a row for every sequence")
    lens = _int32(cache_seqlens, "cache_seqlens", B)
    capacity = max_pages * pool.page_size
    max_k = capacity if max_seqlen_k is None else min(int(max_seqlen_k), capacity)
    w = key_weights
    if w.dtype != torch.float32 or not w.is_cuda or w.dim() != 3 or w.shape[:2] != (B, pool.kv_heads) or \
            w.shape[2] < max_k or w.stride(2) != 1:
        raise ValueError(f"key_weights must be CUDA fp32 [{B}, {pool.kv_heads}, >= {max_k}] with unit stride in its "
                         "last dim")
    if heads is None:
        heads = pool.kv_heads if pool.graph_heads < pool.kv_heads else pool.graph_heads
        _want(heads % pool.kv_heads == 0 and pool.graph_heads in (0, heads),
              "give `heads`: some query heads carry no bias")
    cap_out = table_out.shape[1] * pool.page_size
    budget = int(budget)
    kept = torch.empty((B, pool.kv_heads, max(budget, 0)), dtype=torch.int32, device=w.device)
    lens_out = torch.empty(B, dtype=torch.int32, device=w.device)
    w_out = torch.empty((B, pool.kv_heads, cap_out), dtype=torch.float32, device=w.device)
    a = _lib.Fna2EvictArgs(B, heads, max_k, max_pages, table_out.shape[1], budget, sink, recent, table.data_ptr(),
                           table.stride(0), table_out.data_ptr(), table_out.stride(0), lens.data_ptr(), w.data_ptr(),
                           w.stride(0), w.stride(1), kept.data_ptr(), lens_out.data_ptr(), w_out.data_ptr())
    rc = _lib.load().fna2_evict(pool._ref, ctypes.byref(a), _stream(w.device))
    if rc:
        _lib.check(rc, "fna2_evict")
    return kept, lens_out, w_out
