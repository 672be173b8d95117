"""CPU tests of the paged-cache operators' device checks, with stand-ins for tensors of two
GPUs: every tensor of a call has to lie on the pool's device, and the call is made with that
device current.  Nothing reaches the library."""
import contextlib
import types

import pytest
import torch

from fna2_b200 import _lib, paged

HERE, OTHER = torch.device("cuda", 0), torch.device("cuda", 1)


class Stand:
    """What the Python layer asks of a contiguous tensor."""

    def __init__(self, *shape, dtype=torch.bfloat16, device=HERE):
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, device, True

    def get_device(self):
        return self.device.index

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i=None):
        s = torch.empty(self.shape, device="meta").stride()
        return s if i is None else s[i]

    def data_ptr(self):
        return 4096

    def is_contiguous(self):
        return True

    def contiguous(self):
        return self


def _module(**kw):
    return types.SimpleNamespace(**kw)


T, B, H, KV, D, R = 3, 2, 4, 2, 64, 16


def _pool(**at):
    p = lambda h, c, n: Stand(8, 16, h, c, device=at.get(n, HERE))  # noqa: E731
    return paged.PagedKV(p(KV, D, "k"), p(KV, D, "v"), p(H, R, "rk"))


I32, F32 = torch.int32, torch.float32
CALLS = {
    "append": (paged.qk_norm_rope_append, dict(
        q=(T, H, D), k=(T, KV, D), v=(T, KV, D), r_k=(T, H, R), page_table=(B, 4, I32), cache_seqlens=(B, I32),
        cu_seqlens=(B + 1, I32), positions=(B, I32))),
    "attention": (paged.flash_naylis_paged, dict(
        q=(T, H, D), r_q=(T, H, R), page_table=(B, 4, I32), cache_seqlens=(B, I32), cu_seqlens_q=(B + 1, I32),
        graph_scale=(H, F32), key_weights=(B, KV, 64, F32))),
    "weights": (paged.naylis_key_weights, dict(
        q=(T, H, D), lse=(H, T, F32), r_q=(T, H, R), page_table=(B, 4, I32), cache_seqlens=(B, I32),
        cu_seqlens_q=(B + 1, I32), graph_scale=(H, F32), key_weights=(B, KV, 64, F32))),
    "evict": (paged.naylis_evict, dict(
        key_weights=(B, KV, 64, F32), page_table=(B, 4, I32), cache_seqlens=(B, I32), page_table_out=(B, 1, I32))),
}
MORE = {"append": {}, "attention": dict(max_seqlen_q=2), "weights": dict(max_seqlen_q=2),
        "evict": dict(budget=8, heads=H)}


def _args(call, other=None):
    a = dict(MORE[call], pool=_pool())
    for name, spec in CALLS[call][1].items():
        dtype = spec[-1] if isinstance(spec[-1], torch.dtype) else torch.bfloat16
        shape = spec[:-1] if isinstance(spec[-1], torch.dtype) else spec
        a[name] = Stand(*shape, dtype=dtype, device=OTHER if name == other else HERE)
    return a


@pytest.fixture
def library(monkeypatch):
    """Records (current device, entry) of every call that would reach the library."""
    seen, current = [], [0]

    class Library:
        def __getattr__(self, name):
            def call(*args):
                if not name.endswith("_size"):
                    seen.append((current[0], name))
                return 0
            return call

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d
        yield
        current[0] = before

    real = {n: getattr(torch, n) for n in ("empty", "empty_like")}
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: real["empty"](*a, **{**k, "device": "cpu"}))
    monkeypatch.setattr(torch, "empty_like", lambda t: Stand(*t.shape, dtype=t.dtype, device=t.device))
    return seen, current


@pytest.mark.parametrize("call,name", [(c, n) for c in CALLS for n in CALLS[c][1]])
def test_tensors_of_another_gpu_are_refused(library, call, name):
    with pytest.raises(ValueError, match="pool's device"):
        CALLS[call][0](**_args(call, name))
    assert library[0] == []


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
def test_norm_weights_of_another_gpu_are_refused(library, which):
    norms = {n: _module(weight=Stand(D, dtype=F32, device=OTHER if n == which else HERE), eps=1e-6)
             for n in ("q_norm", "k_norm")}
    with pytest.raises(ValueError, match="pool's device"):
        paged.qk_norm_rope_append(**_args("append"), **norms)
    assert library[0] == []


@pytest.mark.parametrize("which", ["v", "rk"])
def test_a_pool_lies_on_one_device(which):
    with pytest.raises(ValueError, match="pool's device"):
        _pool(**{which: OTHER})


@pytest.mark.parametrize("call", sorted(CALLS))
@pytest.mark.parametrize("current", [0, 1])
def test_the_pools_device_is_current_during_the_call(library, call, current):
    seen, now = library
    now[0] = current
    CALLS[call][0](**_args(call))
    assert len(seen) == 1 and seen[0][0] == 0 and now[0] == current
