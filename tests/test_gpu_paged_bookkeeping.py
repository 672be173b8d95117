"""GPU tests of NaylisPagedCache's bookkeeping: refused calls leave it as it was, attention
belongs to the last append, and no call waits for the device."""
import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_paged import _close_out
from test_gpu_paged_cache import _cache, _tokens

pytestmark = pytest.mark.gpu


def _state(c):
    return (c.free_pages, list(c._free), [list(p) for p in c._pages], list(c.lengths), c.seqlens.tolist(),
            c.positions.tolist(), None if c.key_weights is None else c.key_weights.clone())


def _same(a, b):
    return a[:-1] == b[:-1] and torch.equal(a[-1], b[-1])


def _fill(cache, lens, seed=3):
    q, k, v, rq, rk = _tokens(sum(lens), seed)
    return cache.append(q, k, v, lens, rk), rq


@pytest.mark.parametrize("budget,recent,sink", [(48, 40, 9), (48, -1, 0), (48, 0, -1), (0, 0, 0), (-3, 0, 0)])
def test_a_refused_evict_changes_nothing(budget, recent, sink):
    cache = _cache()
    q, rq = _fill(cache, [100, 20, 65])
    cache.attend(q, rq, torch.randn(4, device="cuda"))
    before = _state(cache)
    for _ in range(3):
        with pytest.raises((RuntimeError, ValueError)):
            cache.evict(budget, recent, sink)
    assert _same(_state(cache), before)
    assert cache.evict(48, 8, 2) == [0, 2] and cache.lengths == [48, 20, 48]


def test_a_refused_append_changes_nothing():
    cache = _cache()
    q0, rq0 = _fill(cache, [30, 20, 5])
    gs = torch.randn(4, device="cuda")
    first = cache.attend(q0, rq0, gs, weigh=False)
    before = _state(cache)
    q, k, v, _, rk = _tokens(90, 4)
    for bad in (dict(r_k=None), dict(k=k.float()), dict(v=v[:, :1]), dict(q_norm=torch.nn.Identity())):
        with pytest.raises((RuntimeError, ValueError, TypeError, AttributeError)):
            cache.append(**{**dict(q=q, k=k, v=v, new=[70, 0, 20], r_k=rk), **bad})
    assert _same(_state(cache), before)
    assert torch.equal(cache.attend(q0, rq0, gs, weigh=False), first)  # still the tokens of the last append


def test_attend_takes_the_tokens_of_the_last_append():
    cache = _cache()
    gs = torch.randn(4, device="cuda")
    q, _, _, rq, _ = _tokens(6, 5)
    with pytest.raises(ValueError, match="last append"):
        cache.attend(q, rq, gs)
    qa, rqa = _fill(cache, [30, 20, 5])
    with pytest.raises(ValueError, match="last append"):
        cache.attend(q, rq, gs)
    assert torch.isfinite(cache.attend(qa, rqa, gs)).all()


@pytest.mark.parametrize("gone", [0, 2])
def test_attend_after_a_release(gone):
    """The released slot's tokens see no key, the others what they saw."""
    from fna2_b200 import _lib
    cache = _cache()
    gs = torch.randn(4, device="cuda")
    new = [90, 3, 20]
    q, rq = _fill(cache, new)
    want, wl = cache.attend(q, rq, gs, weigh=False, return_lse=True)
    cache.release(gone)
    out, lse = cache.attend(q, rq, gs, weigh=False, return_lse=True)
    torch.cuda.synchronize()
    assert _lib.load().fna2_device_status(1) == 0
    for b, (o, w, l, m) in enumerate(zip(out.split(new), want.split(new), lse.split(new, 1), wl.split(new, 1))):
        if b == gone:
            assert (o == 0).all() and torch.isneginf(l).all()
        else:
            assert (o.float() - w.float()).abs().max() <= 2.0 ** -7 * w.float().abs().max()
            assert torch.allclose(l, m, atol=30 * 2.0 ** -16 + 2e-5)


def test_attend_after_an_evict():
    """As long as the eviction kept the last tokens' own keys; not when it took some."""
    for recent, ok in ((3, True), (2, False)):
        cache = _cache()
        gs = torch.randn(4, device="cuda")
        q, rq = _fill(cache, [100, 20, 65])
        cache.attend(q, rq, gs)
        q, k, v, rq, rk = _tokens(9, 8)
        q = cache.append(q, k, v, [3, 3, 3], rk)
        cache.attend(q, rq, gs)
        cut = cache.evict(48, recent, 2)
        assert cut == [0, 2]
        if ok:
            x = dict(kp=cache.pool.k_pages.cpu(), vp=cache.pool.v_pages.cpu(), rp=cache.pool.rk_pages.cpu(),
                     table=cache.page_table.cpu(), lens=cache.lengths, cu=torch.tensor([0, 3, 6, 9]), q=q.cpu(),
                     rq=rq.cpu(), gs=gs.cpu())
            _close_out("after evict", cache.attend(q, rq, gs), PO.attention(x, True)[0])
            continue
        with pytest.raises(RuntimeError, match="before evict"):
            cache.attend(q, rq, gs)
        cache.release(0)
        with pytest.raises(RuntimeError, match="before evict"):
            cache.attend(q, rq, gs)
        q, k, v, rq, rk = _tokens(3, 9)
        assert torch.isfinite(cache.attend(cache.append(q, k, v, [1, 1, 1], rk), rq, gs)).all()


def test_no_call_waits_for_the_device():
    """Appends that take pages (all slots one token, or different numbers), attention, eviction and release
    return while the device is still busy with what came before."""
    cache = _cache(num_pages=60)
    gs = torch.randn(4, device="cuda")
    steps = [[100, 31, 64], [1, 1, 1], [12, 0, 16], [1, 1, 1]]
    data = [_tokens(sum(new), 20 + i) for i, new in enumerate(steps)]

    def serve(c):
        outs = []
        for new, (q, k, v, rq, rk) in zip(steps, data):
            q = c.append(q, k, v, new, rk)
            outs.append(c.attend(q, rq, gs))
        c.evict(48, 16, 2)
        c.release(1)
        q, k, v, rq, rk = data[1]
        outs.append(c.attend(c.append(q, k, v, [1, 1, 1], rk), rq, gs))
        return outs
    want = serve(_cache(num_pages=60))  # (and the library, its kernels and the allocators' blocks are there)
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    done = torch.cuda.Event()
    torch.cuda.set_sync_debug_mode("error")
    try:
        torch.cuda._sleep(2 ** 30)  # about half a second
        done.record()
        got = serve(cache)
        busy = not done.query()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    torch.cuda.synchronize()
    assert busy
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    assert cache.page_table[1].tolist()[:1] != [-1] and cache.seqlens.tolist() == cache.lengths
