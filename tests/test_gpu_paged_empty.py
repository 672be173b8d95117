"""GPU tests of the paged-cache operators on nothing: no sequence, no new token, no page."""
import pytest
import torch

from test_gpu_paged import _make, _pool, _status

pytestmark = pytest.mark.gpu


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rows(n, h, c):
    return torch.ones(n, h, c, dtype=torch.bfloat16, device="cuda")


@pytest.mark.parametrize("batch", [0, 3])
def test_no_sequence_and_no_page(batch):
    """A step without a sequence; sequences that own no page yet (queries of theirs see no key)."""
    from fna2_b200.paged import flash_naylis_paged, naylis_evict, naylis_key_weights, qk_norm_rope_append
    pool = _pool(_make([40], [1], 4, 2, 4, 64, 16, 16, 1))
    table = torch.empty(batch, 0, dtype=torch.int32, device="cuda")
    lens, cu = _ints(*[0] * batch), _ints(*range(batch + 1))
    q, rq, gs = _rows(batch, 4, 64), _rows(batch, 4, 16), torch.ones(4, device="cuda")
    out, lse = flash_naylis_paged(q, pool, table, lens, cu, 1, r_q=rq, graph_scale=gs, return_lse=True)
    assert out.shape == (batch, 4, 64) and (out == 0).all() and torch.isneginf(lse).all()
    w = naylis_key_weights(q, lse, pool, table, lens, cu, 1, r_q=rq, graph_scale=gs)
    assert w.shape == (batch, 2, 0)
    kept, n, wo = naylis_evict(w, pool, table, lens, 8, torch.zeros(batch, 1, dtype=torch.int32, device="cuda"), heads=4)
    assert (kept == -1).all() and n.tolist() == [0] * batch and (wo == 0).all()
    k0 = pool.k_pages.clone()
    none = _ints(*[0] * (batch + 1))
    o = qk_norm_rope_append(_rows(0, 4, 64), _rows(0, 2, 64), _rows(0, 2, 64), pool, table, lens, none, r_k=_rows(0, 4, 16))
    assert o.shape == (0, 4, 64) and torch.equal(pool.k_pages.view(torch.int16), k0.view(torch.int16))
    assert _status() == 0
