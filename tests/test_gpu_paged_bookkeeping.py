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
