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
631 append, 641 attention and key weights, 651 eviction).  So is a page id outside
the pool: append and eviction do not write its rows, the others read them as zeros.

NaylisPagedCache keeps the pool, the tables and the lengths, and runs the four.

These are calls for inference: results carry no gradient, whether or not the inputs
require one (as in flash_naylis_decode), and pools and key weights are written in place
without autograd or torch.compile knowing of it (call them outside compiled regions).
Every tensor of a call lies on the pool's device; the work goes to that device's
current stream.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib

_DT = {torch.float32: _lib.FNA2_DTYPE_F32, torch.bfloat16: _lib.FNA2_DTYPE_BF16}

# The argument blocks of include/fna2.h, packed in one call each: filling a ctypes structure field
# by field costs several microseconds, as much as a small kernel.
_ATTN_ARGS = struct.Struct("@8if PqPP PqqPqqP Pqq Pq Pqqq".replace(" ", ""))
_APPEND_ARGS = struct.Struct("@6iq PqqPqqPqqPqqPqq Pq PPP PP f P".replace(" ", ""))
_EVICT_ARGS = struct.Struct("@8i PqPqP Pqq PPP".replace(" ", ""))


def _want(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


# Every tensor of a call lies on the pool's device (`gpu`: its index): a kernel takes pointers as they are.
def _elsewhere(t: torch.Tensor, name: str, gpu: int) -> ValueError:
    return ValueError(f"{name} must be a CUDA tensor on the pool's device cuda:{gpu} (got {t.device})")


def _rows(t: torch.Tensor, name: str, tokens: int, heads: int, cols: int, dtype: torch.dtype, gpu: int):
    """Checks a [tokens, heads, cols] tensor; returns it with its pointer and token and head
    strides.  Rows that are not 16-byte aligned or columns without unit stride are copied once."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if t.shape != (tokens, heads, cols):
        raise ValueError(f"{name} must be [{tokens}, {heads}, {cols}] (got {tuple(t.shape)})")
    if t.get_device() != gpu:
        raise _elsewhere(t, name, gpu)
    s0, s1, s2 = t.stride()
    p = t.data_ptr()
    if s2 != 1 or p & 15 or ((s0 | s1) * (2 if dtype is torch.bfloat16 else 4)) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.data_ptr(), heads * cols, cols
    return t, p, s0, s1


def _int32(t: torch.Tensor, name: str, n: int, gpu: int) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.numel() != n:
        raise ValueError(f"{name} must be a CUDA int32 tensor of {n} entries")
    if t.get_device() != gpu:
        raise _elsewhere(t, name, gpu)
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, gpu: int, name: str = "page_table") -> torch.Tensor:
    if t.dtype is not torch.int32 or t.dim() != 2:
        raise ValueError(f"{name} must be a CUDA int32 tensor [batch, pages]")
    if t.get_device() != gpu:
        raise _elsewhere(t, name, gpu)
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _empty(like: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(like) if like.is_contiguous() else torch.empty(like.shape, dtype=like.dtype,
                                                                           device=like.device)


def _launch(gpu: int, call, *args) -> int:
    """call(*args, the GPU's current stream) with that GPU current, where the kernels go."""
    if torch._C._cuda_getDevice() == gpu:
        return call(*args, torch._C._cuda_getCurrentRawStream(gpu))  # current_stream().cuda_stream, without the object
    with torch.cuda.device(gpu):
        return call(*args, torch._C._cuda_getCurrentRawStream(gpu))


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
            if t.get_device() != k_pages.get_device():
                raise _elsewhere(t, name, k_pages.get_device())
            _want(t.dim() == 4, f"{name} must be [pages, page_size, heads, columns] (got {tuple(t.shape)})")
            _want(t.stride(3) == 1, f"{name} must have unit stride in its last dim")
            _want(t.shape[:2] == k_pages.shape[:2], f"{name} must have the pages and page size of k_pages")
        _want(v_pages.shape == k_pages.shape, "v_pages must have the shape of k_pages")
        self.k_pages, self.v_pages, self.rk_pages = k_pages, v_pages, rk_pages
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = k_pages.shape
        self.graph_heads, self.rank = (0, 16) if rk_pages is None else rk_pages.shape[2:]
        if self.graph_heads == 0:
            rk_pages = None
        self.device, self.gpu = k_pages.device, k_pages.get_device()
        c = _lib.Fna2PagedKV(self.num_pages, self.page_size, self.kv_heads, self.graph_heads, self.head_dim, self.rank)
        c.k, c.v = k_pages.data_ptr(), v_pages.data_ptr()
        c.k_page_stride, c.k_token_stride, c.k_head_stride = k_pages.stride()[:3]
        c.v_page_stride, c.v_token_stride, c.v_head_stride = v_pages.stride()[:3]
        if rk_pages is not None:
            c.rk = rk_pages.data_ptr()
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
    dt = q.dtype
    if dt not in _DT:
        raise TypeError(f"q must be fp32 or bf16 (got {dt})")
    _want(q.dim() == 3, f"q must be [T, H, D] (got {tuple(q.shape)})")
    (T, H, D), gpu = q.shape, pool.gpu
    q, q_p, q_0, q_1 = _rows(q, "q", T, H, pool.head_dim, dt, gpu)
    k, k_p, k_0, k_1 = _rows(k, "k", T, pool.kv_heads, D, dt, gpu)
    v, v_p, v_0, v_1 = _rows(v, "v", T, pool.kv_heads, D, dt, gpu)
    _want((r_k is not None) == (pool.graph_heads > 0), "r_k goes with a pool that has rk_pages")
    r_p = r_0 = r_1 = 0
    if r_k is not None:
        r_k, r_p, r_0, r_1 = _rows(r_k, "r_k", T, pool.graph_heads, pool.rank, dt, gpu)
    table = _table(page_table, gpu)
    B, max_pages = table.shape
    lens, cu = _int32(cache_seqlens, "cache_seqlens", B, gpu), _int32(cu_seqlens, "cu_seqlens", B + 1, gpu)
    if positions is not None:
        positions = _int32(positions, "positions", B, gpu)
    _want((q_norm is None) == (k_norm is None), "give both norms or neither")
    wq_p = wk_p = f_p = 0
    eps, w_dt, rope_dt = 0.0, 0, _DT[dt]
    if q_norm is not None:
        wq, wk, eps = q_norm.weight, k_norm.weight, float(q_norm.eps)
        _want(wq.dtype in _DT and wk.dtype == wq.dtype and wq.numel() == D and wk.numel() == D,
              "norm weights: CUDA fp32 or bf16 [head_dim], same dtype")
        for w, name in ((wq, "q_norm.weight"), (wk, "k_norm.weight")):
            if w.get_device() != gpu:
                raise _elsewhere(w, name, gpu)
        _want(eps == float(k_norm.eps), "the two norms must share eps")
        wq, wk = wq.contiguous(), wk.contiguous()
        wq_p, wk_p, w_dt, rope_dt = wq.data_ptr(), wk.data_ptr(), _DT[wq.dtype], _DT[torch.promote_types(dt, wq.dtype)]
    if rope is not None:
        f = rope.inv_freq
        if f.dtype is not torch.float32 or f.device != q.device or not f.is_contiguous():
            f = f.detach().to(device=q.device, dtype=torch.float32).contiguous()
        _want(f.numel() == D // 2, "rope.inv_freq must have head_dim / 2 entries")
        f_p = f.data_ptr()
    out = _empty(q) if dt is torch.bfloat16 else torch.empty((T, H, D), dtype=torch.bfloat16, device=q.device)
    a = _APPEND_ARGS.pack(B, H, max_pages, _DT[dt], w_dt, rope_dt, T, q_p, q_0, q_1, k_p, k_0, k_1, v_p, v_0, v_1, r_p,
                          r_0, r_1, out.data_ptr(), H * D, D, table.data_ptr(), table.stride(0), lens.data_ptr(),
                          cu.data_ptr(), 0 if positions is None else positions.data_ptr(), wq_p, wk_p, eps, f_p)
    rc = _launch(gpu, _lib.load().fna2_paged_append, pool._ref, a)
    if rc:
        _lib.check(rc, "fna2_paged_append")
    return out


def _weights_ok(w: torch.Tensor, B: int, heads: int, keys: int, gpu: int) -> None:
    if w.dtype is not torch.float32 or w.dim() != 3 or w.shape[0] != B or w.shape[1] != heads or \
            w.shape[2] < keys or w.stride(2) != 1:
        raise ValueError(f"key_weights must be CUDA fp32 [{B}, {heads}, >= {keys}] with unit stride in its last dim")
    if w.get_device() != gpu:
        raise _elsewhere(w, "key_weights", gpu)


def _attention(name, q, pool, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, r_q, graph_scale, softmax_scale,
               is_causal, key_weights, max_seqlen_k, num_splits, out, lse, clear=0):
    """Packs the arguments of fna2_paged_attn or fna2_key_weights and calls it."""
    (T, H, D), gpu = q.shape, pool.gpu
    q, q_p, q_0, q_1 = _rows(q, "q", T, H, pool.head_dim, torch.bfloat16, gpu)
    table = _table(page_table, gpu)
    B, max_pages = table.shape
    lens, cu = _int32(cache_seqlens, "cache_seqlens", B, gpu), _int32(cu_seqlens_q, "cu_seqlens_q", B + 1, gpu)
    max_k = max_pages * pool.page_size
    if max_seqlen_k is not None and max_seqlen_k < max_k:
        max_k = int(max_seqlen_k)
    r_p = r_0 = r_1 = gs_p = 0
    if pool.graph_heads:
        _want(r_q is not None and graph_scale is not None, "graph heads need r_q and graph_scale")
        r_q, r_p, r_0, r_1 = _rows(r_q, "r_q", T, pool.graph_heads, pool.rank, torch.bfloat16, gpu)
        gs = graph_scale
        _want(gs.numel() == pool.graph_heads, "graph_scale must be a CUDA tensor [H_G]")
        if gs.get_device() != gpu:
            raise _elsewhere(gs, "graph_scale", gpu)
        if gs.dtype is not torch.float32 or not gs.is_contiguous():
            gs = gs.detach().float().contiguous()
        gs_p = gs.data_ptr()
    else:
        _want(r_q is None, "r_q goes with a pool that has rk_pages")
    w_p = w_0 = w_1 = 0
    if key_weights is not None:
        _weights_ok(key_weights, B, pool.kv_heads, max_k, gpu)
        w_p, (w_0, w_1, _) = key_weights.data_ptr(), key_weights.stride()
    l_p, l_0 = (0, 0) if lse is None else (lse.data_ptr(), lse.stride(0))
    a = _ATTN_ARGS.pack(B, H, T, int(max_seqlen_q), max_k, max_pages, 1 if is_causal else 0, num_splits,
                        D ** -0.5 if softmax_scale is None else softmax_scale, table.data_ptr(), table.stride(0),
                        lens.data_ptr(), cu.data_ptr(), q_p, q_0, q_1, r_p, r_0, r_1, gs_p,
                        0 if out is None else out.data_ptr(), H * D, D, l_p, l_0, w_p, w_0, w_1, clear)
    lib = _lib.load()
    size, call = ((lib.fna2_paged_attn_workspace_size, lib.fna2_paged_attn) if out is not None else
                  (lib.fna2_key_weights_workspace_size, lib.fna2_key_weights))
    n, ws_p = size(pool._ref, a), 0
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=pool.device)
        ws_p = ws.data_ptr()
    rc = _launch(gpu, call, pool._ref, a, ws_p, n)
    if rc:
        _lib.check(rc, name)


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
    _want(q.dim() == 3, f"q must be [T, H, D] (got {tuple(q.shape)})")
    T, H, D = q.shape
    out = _empty(q)
    lse = torch.empty((H, T), dtype=torch.float32, device=q.device) if return_lse else None
    _attention("fna2_paged_attn", q, pool, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, r_q, graph_scale,
               softmax_scale, is_causal, key_weights, max_seqlen_k, num_splits, out, lse)
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
    _want(q.dim() == 3, f"q must be [T, H, D] (got {tuple(q.shape)})")
    if lse.dtype is not torch.float32 or lse.shape != (q.shape[1], q.shape[0]):
        raise ValueError(f"lse must be CUDA fp32 [{q.shape[1]}, {q.shape[0]}] (got {lse.dtype} {tuple(lse.shape)})")
    if lse.get_device() != pool.gpu:
        raise _elsewhere(lse, "lse", pool.gpu)
    if lse.stride(1) != 1:
        lse = lse.contiguous()
    clear = 0
    if key_weights is None:
        clear = page_table.shape[1] * pool.page_size
        key_weights = torch.empty((page_table.shape[0], pool.kv_heads, clear), dtype=torch.float32, device=q.device)
    _attention("fna2_key_weights", q, pool, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, r_q, graph_scale,
               softmax_scale, is_causal, key_weights, max_seqlen_k, 0, None, lse, clear)
    return key_weights


def naylis_evict(key_weights: torch.Tensor, pool: PagedKV, page_table: torch.Tensor, cache_seqlens: torch.Tensor,
                 budget: int, page_table_out: torch.Tensor, heads: int, recent: int = 0, sink: int = 0,
                 max_seqlen_k: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keep, per sequence and KV head, min(len, budget) keys: the first `sink`, the last
    `recent`, and of the others those of the largest key_weights [B, H_KV, >= max_seqlen_k]
    (ties to the lowest index, NaN below every number).  Their rows of K, V and R_k are copied
    in order to slots [0, kept) of the pages of page_table_out [B, >= budget / page_size], which
    must be pages that no sequence of the call occupies; the old pages are the caller's to
    free.  heads: query heads (R_k moves with the KV head of its query head).
    Returns kept [B, H_KV, budget] int32 (-1 past the count), the new lengths [B] int32, and the
    kept keys' weights [B, H_KV, pages_out * page_size] (0 past the count)."""
    dev, gpu = pool.device, pool.gpu
    table, table_out = _table(page_table, gpu), _table(page_table_out, gpu, "page_table_out")
    B, max_pages = table.shape
    pages_out = table_out.shape[1]
    _want(table_out.shape[0] == B, "page_table_out must have a row for every sequence")
    lens = _int32(cache_seqlens, "cache_seqlens", B, gpu)
    max_k = max_pages * pool.page_size
    if max_seqlen_k is not None and max_seqlen_k < max_k:
        max_k = int(max_seqlen_k)
    _weights_ok(key_weights, B, pool.kv_heads, max_k, gpu)
    w_0, w_1, _ = key_weights.stride()
    kept = torch.empty((B, pool.kv_heads, max(budget, 0)), dtype=torch.int32, device=dev)
    lens_out = torch.empty_like(lens)
    w_out = torch.empty((B, pool.kv_heads, pages_out * pool.page_size), dtype=torch.float32, device=dev)
    a = _EVICT_ARGS.pack(B, heads, max_k, max_pages, pages_out, budget, sink, recent, table.data_ptr(), table.stride(0),
                         table_out.data_ptr(), table_out.stride(0), lens.data_ptr(), key_weights.data_ptr(), w_0, w_1,
                         kept.data_ptr(), lens_out.data_ptr(), w_out.data_ptr())
    rc = _launch(gpu, _lib.load().fna2_evict, pool._ref, a)
    if rc:
        _lib.check(rc, "fna2_evict")
    return kept, lens_out, w_out


class NaylisPagedCache:
    """The paged cache of one layer: a pool, and per batch slot its pages, length, next rotary
    position and key weights.

    Lengths are kept on the host (they follow from the calls) and on the device, and what the
    host decides goes there from pinned memory, so no call waits for the device.  A slot's pages are taken from a free list as it grows; evict moves
    what it keeps to fresh pages and returns the old ones.  All work is ordered by the current
    stream; pages that are returned are reused by later calls on the same stream.

        cache = NaylisPagedCache(pages, 64, batch, 32768, H, H_KV, D, graph_heads=H_G, rank=R)
        q = cache.append(q, k, v, new, r_k, q_norm, k_norm, rope)     # new[b] tokens for slot b
        out = cache.attend(q, r_q, graph_scale)                       # the tokens just appended
        cache.evict(budget=4096, recent=256, sink=4)
    """

    def __init__(self, num_pages: int, page_size: int, batch: int, max_len: int, heads: int, kv_heads: int,
                 head_dim: int, graph_heads: int = 0, rank: int = 16, key_weights: bool = True, device="cuda"):
        def pages(h, c):
            return torch.zeros(num_pages, page_size, h, c, device=device, dtype=torch.bfloat16)
        self.pool = PagedKV(pages(kv_heads, head_dim), pages(kv_heads, head_dim),
                            pages(graph_heads, rank) if graph_heads else None)
        self.heads, self.batch, self.page_size = heads, batch, page_size
        self.max_pages = -(-max_len // page_size)
        dev = self.pool.device
        self.page_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=dev)
        self.seqlens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.positions = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.key_weights = (torch.zeros(batch, kv_heads, self.max_pages * page_size, device=dev) if key_weights
                            else None)
        self.lengths: List[int] = [0] * batch
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(num_pages))[::-1]
        self._new: List[int] = [0] * batch  # tokens of the last append
        self._evicted: List[int] = []       # slots that have lost some of them since
        self._cu = torch.zeros(batch + 1, dtype=torch.int32, device=dev)
        self._one_each = torch.arange(batch + 1, dtype=torch.int32, device=dev)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _send(self, values: Sequence[int], dtype=torch.int64) -> torch.Tensor:
        """Integers to the device, in stream order and without a wait (pinned memory is kept until it is copied)."""
        return torch.tensor(values, dtype=dtype, pin_memory=True).to(self.pool.device, non_blocking=True)

    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise RuntimeError(f"the pool has {len(self._free)} free pages, {n} are needed")
        taken, self._free = self._free[len(self._free) - n:], self._free[:len(self._free) - n]
        return taken[::-1]

    def _grow(self, new: Sequence[int]) -> List[int]:
        """Pages for new[b] more tokens of each slot; returns how many each slot got."""
        need = [max(0, -(-(n + m) // self.page_size) - len(p)) for n, m, p in zip(self.lengths, new, self._pages)]
        for b, (n, m) in enumerate(zip(self.lengths, new)):
            _want(m >= 0 and -(-(n + m) // self.page_size) <= self.max_pages,
                  f"slot {b}: {n} + {m} tokens do not fit its {self.max_pages} pages")
        taken = self._take(sum(need))
        at, places = 0, []
        for b, x in enumerate(need):
            first = b * self.max_pages + len(self._pages[b])
            places += range(first, first + x)
            self._pages[b] += taken[at:at + x]
            at += x
        if taken:  # one copy and one launch, however many slots take pages
            entries = self._send(places + taken)
            self.page_table.view(-1).index_copy_(0, entries[:at], entries[at:].int())
        return need

    def _shrink(self, got: Sequence[int]) -> None:
        """Takes back what _grow gave."""
        for b in reversed(range(self.batch)):
            if got[b]:
                self._free += self._pages[b][:-got[b] - 1:-1]
                del self._pages[b][-got[b]:]

    def append(self, q, k, v, new: Sequence[int], r_k=None, q_norm=None, k_norm=None, rope=None) -> torch.Tensor:
        """new[b] new tokens of every slot b (0 for none), packed in slot order: q, k through the
        norms and the rotary embedding, k, v, r_k into the pages (qk_norm_rope_append).  Returns
        q for attend()."""
        new = [int(n) for n in new]
        _want(len(new) == self.batch and sum(new) == q.shape[0], "new must give the tokens of every slot")
        got = self._grow(new)
        try:
            ones = all(n == 1 for n in new)
            if ones:
                cu = self._one_each
            else:
                starts = [0]
                for n in new:
                    starts.append(starts[-1] + n)
                cu = self._send(starts, torch.int32)
            out = qk_norm_rope_append(q, k, v, self.pool, self.page_table, self.seqlens, cu, r_k, self.positions,
                                      q_norm, k_norm, rope)
        except Exception:
            self._shrink(got)
            raise
        self._cu, self._evicted = cu, []
        added = 1 if ones else self._cu[1:] - self._cu[:-1]
        self.seqlens += added
        self.positions += added
        self.lengths = [a + b for a, b in zip(self.lengths, new)]
        self._new = new
        return out

    def attend(self, q, r_q=None, graph_scale=None, softmax_scale=None, weigh: bool = True, return_lse: bool = False):
        """Attention of the tokens of the last append over their slots' keys (flash_naylis_paged);
        weigh: add the attention weights to key_weights.  Slots that were released since have no
        keys: 0 and -inf.  An evict that took some of these tokens' own keys away comes after it."""
        _want(q.dim() == 3 and q.shape[0] == sum(self._new), "attend takes the tokens of the last append")
        if self._evicted:
            raise RuntimeError(f"slots {self._evicted}: tokens of the last append were evicted, attend comes before evict")
        return flash_naylis_paged(q, self.pool, self.page_table, self.seqlens, self._cu, max(self._new), r_q,
                                  graph_scale, softmax_scale, True, self.key_weights if weigh else None, return_lse,
                                  max(self.lengths))

    def evict(self, budget: int, recent: int = 0, sink: int = 0) -> List[int]:
        """Cut every slot with more than `budget` keys to `budget` (naylis_evict).  Rotary positions
        go on from where they were.  Returns the slots that were cut."""
        _want(self.key_weights is not None, "evict needs a cache with key weights")
        over = [b for b, n in enumerate(self.lengths) if n > budget]
        if not over:
            return over
        per = -(-budget // self.page_size)
        fresh = self._take(per * len(over))
        rows = [fresh[i * per:(i + 1) * per] for i in range(len(over))]
        try:
            sent = self._send(over + fresh)
            idx, table_out = sent[:len(over)], sent[len(over):].view(len(over), per).int()
            _, lens, w = naylis_evict(self.key_weights[idx], self.pool, self.page_table[idx], self.seqlens[idx], budget,
                                      table_out, self.heads, recent, sink, max(self.lengths))
        except Exception:
            self._free += fresh[::-1]
            raise
        self.page_table.index_fill_(0, idx, -1)
        self.page_table[:, :per].index_copy_(0, idx, table_out)
        self.seqlens.index_copy_(0, idx, lens)
        self.key_weights.index_fill_(0, idx, 0.0)
        self.key_weights[:, :, :w.shape[2]].index_copy_(0, idx, w)
        for b, row in zip(over, rows):
            self._free += self._pages[b]
            self._pages[b] = list(row)
            self.lengths[b] = budget
        self._evicted += [b for b in over if recent < self._new[b]]
        return over

    def release(self, slot: int) -> None:
        """Empty a slot; its pages go back to the pool."""
        self._free += self._pages[slot]
        self._pages[slot], self.lengths[slot] = [], 0
        self._evicted = [b for b in self._evicted if b != slot]
        self.page_table[slot].fill_(-1)  # (assigning a number copies it from the host)
        self.seqlens[slot].zero_()
        self.positions[slot].zero_()
        if self.key_weights is not None:
            self.key_weights[slot].zero_()
