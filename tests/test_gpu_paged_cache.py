"""GPU tests of NaylisPagedCache and of the serving example: the cache's bookkeeping against
what the operators give on plain tensors, and the whole path end to end."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cache(**kw):
    from fna2_b200.paged import NaylisPagedCache
    a = dict(num_pages=40, page_size=16, batch=3, max_len=256, heads=4, kv_heads=2, head_dim=64, graph_heads=4, rank=16)
    return NaylisPagedCache(**{**a, **kw})


def _tokens(n, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda h, c: torch.randn(n, h, c, generator=g).bfloat16().cuda()  # noqa: E731
    return r(4, 64), r(2, 64), r(2, 64), r(4, 16), r(4, 16)


def test_chunks_decode_and_release():
    """Any split of a sequence into appends gives the same cache, and attention over it is that
    of the packed op; released pages come back."""
    from fna2_b200 import flash_naylis_attn
    L = [100, 37, 1]
    data = [_tokens(n, 5 + i) for i, n in enumerate(L)]
    gs = torch.randn(4, device="cuda")
    cache = _cache()
    outs, done = [[], [], []], [0, 0, 0]
    for new in ([30, 37, 0], [1, 0, 1], [68, 0, 0], [1, 0, 0]):
        part = [torch.cat([data[b][i][done[b]:done[b] + n] for b, n in enumerate(new)]) for i in range(5)]
        q = cache.append(part[0], part[1], part[2], new, part[4])
        o = cache.attend(q, part[3], gs)
        for b, piece in enumerate(o.split(new)):
            outs[b].append(piece)
        done = [d + n for d, n in zip(done, new)]
    assert cache.lengths == L == cache.seqlens.tolist() == cache.positions.tolist()
    for b in range(3):
        cu = torch.tensor([0, L[b]], dtype=torch.int32, device="cuda")
        ref = flash_naylis_attn(*data[b], gs, is_causal=True, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=L[b],
                                max_seqlen_k=L[b]).float()
        got = torch.cat(outs[b]).float()
        # two kernels of bf16 outputs, each within 2^-8 of the value and of the largest (see test_gpu_paged)
        assert ((got - ref).abs() <= 2.0 ** -6 * (ref.abs() + ref.abs().max())).all()
        # every query gives weight 1 per head, spread over the keys it saw
        assert abs(cache.key_weights[b].sum().item() - 4 * L[b]) <= 1e-3 * L[b]
        assert (cache.key_weights[b, :, L[b]:] == 0).all()
    free = cache.free_pages
    cache.release(0)
    assert cache.free_pages == free + 7 and cache.seqlens.tolist() == [0, 37, 1]


def test_evict_keeps_the_heaviest_and_goes_on():
    cache = _cache()
    L = [100, 20, 65]
    parts = [torch.cat(x) for x in zip(*[_tokens(n, 50 + n) for n in L])]
    q = cache.append(parts[0], parts[1], parts[2], L, parts[4])
    cache.attend(q, parts[3], torch.randn(4, device="cuda"))
    w = cache.key_weights.clone()
    total = 40 - cache.free_pages
    assert total == 7 + 2 + 5
    assert cache.evict(budget=48, recent=8, sink=2) == [0, 2]
    assert cache.lengths == [48, 20, 48] == cache.seqlens.tolist() and cache.positions.tolist() == L
    assert 40 - cache.free_pages == 3 + 2 + 3
    used = [p for row in cache.page_table.tolist() for p in row if p >= 0]
    assert len(set(used)) == len(used) == 8
    for b in (0, 2):
        for h in range(2):
            old = w[b, h, 2:L[b] - 8]
            best = old.topk(38).values.sum() + w[b, h, :2].sum() + w[b, h, L[b] - 8:L[b]].sum()
            assert torch.allclose(cache.key_weights[b, h, :48].sum(), best, rtol=1e-5)
    q, k, v, rq, rk = _tokens(3, 99)
    out = cache.attend(cache.append(q, k, v, [1, 1, 1], rk), rq, torch.randn(4, device="cuda"))
    assert torch.isfinite(out).all() and cache.lengths == [49, 21, 49] and cache.positions.tolist() == [101, 21, 66]


def test_cache_refuses_what_does_not_fit():
    cache = _cache(num_pages=5)
    q, k, v, rq, rk = _tokens(100, 1)
    with pytest.raises(RuntimeError, match="free pages"):
        cache.append(q, k, v, [100, 0, 0], rk)
    with pytest.raises(ValueError, match="every slot"):
        cache.append(q, k, v, [50, 50], rk)
    with pytest.raises(ValueError, match="do not fit"):
        _cache().append(*[torch.zeros(300, h, 64, device="cuda").bfloat16() for h in (4, 2, 2)], [300, 0, 0],
                        torch.zeros(300, 4, 16, device="cuda").bfloat16())
    assert cache.lengths == [0, 0, 0] and cache.free_pages == 5


def test_serving_example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import paged_serving
    got = paged_serving.run(heads=8, kv_heads=2, head_dim=64, rank=32, embed=256, prompts=(700, 33, 260), chunk=200,
                            budget=256, recent=32, steps=6, drafted=3, verbose=False)
    # outputs pass a bf16 projection of 512 terms after two attention kernels of 2^-8 each
    assert got["deviation"] <= 2.0 ** -5
    assert got["lengths"] == got["device_lengths"] == [256, 33 + 6 * 4, 256]
    assert got["positions"] == [700 + 24, 33 + 24, 260 + 24]
