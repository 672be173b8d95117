"""GPU tests of the paged attention with infinities and NaN among the values in use: they reach
the rows that the definition lets them reach, and no others, whichever kernel serves the row.

Tolerances are those of test_gpu_paged (their derivation is there)."""
import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_paged import _close_lse, _close_out, _close_w, _dev, _make, _pool, _status

pytestmark = pytest.mark.gpu


def _attend(x, splits=0, causal=True):
    from fna2_b200.paged import flash_naylis_paged
    d = _dev(x)
    return flash_naylis_paged(d["q"], _pool(x), d["table"], d["lens"], d["cu"], max(x["new"]), r_q=d["rq"],
                              graph_scale=d["gs"], is_causal=causal, return_lse=True, num_splits=splits)


# H, H_KV, H_G, R, new: single rows, several heads or tokens in one block of 16 rows, several blocks, the
# tensor-core kernel
SHAPES = [(4, 2, 4, 16, 1), (8, 2, 8, 32, 3), (8, 2, 6, 24, 2), (16, 2, 11, 8, 5), (8, 1, 8, 16, 7), (4, 2, 4, 32, 140)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_one_heads_r_k_stays_with_that_head(shape, value):
    H, H_KV, H_G, R, new = shape
    x = _make([200], [new], H, H_KV, H_G, 64, R, 32, 31)
    ref, lse, _ = PO.attention(x, True)
    h, key = 1, 20  # every row sees key 20
    page = (int(x["table"][0, key // 32]), key % 32)
    x["rp"][page[0], page[1], h, 3] = value
    out, l2 = _attend(x)
    rest = [i for i in range(H) if i != h]
    _close_out("the other heads", out[:, rest], ref[:, rest])
    _close_lse(l2[rest], lse[rest])
    if value != value:  # every query of that head has a NaN logit
        assert torch.isnan(out[:, h]).all() and torch.isnan(l2[h]).all()


@pytest.mark.parametrize("splits", [1, 5])
@pytest.mark.parametrize("new", [1, 3, 40, 300])
def test_a_query_of_nan_gives_nan(new, splits):
    """All logits of the row are NaN; the other rows are what they were."""
    x = _make([900], [new], 4, 2, 4, 64, 16, 32, 17)
    ref, lse, _ = PO.attention(x, True)
    x["q"][new // 2, 1] = float("nan")
    out, l2 = _attend(x, splits)
    assert torch.isnan(out[new // 2, 1]).all() and torch.isnan(l2[1, new // 2])
    keep = torch.ones(new, 4, dtype=torch.bool)
    keep[new // 2, 1] = False
    _close_out("the others", out.cpu()[keep], ref[keep])
    _close_lse(l2.cpu().t()[keep], lse.t()[keep])


@pytest.mark.parametrize("splits", [1, 9, 70])
@pytest.mark.parametrize("new", [1, 6, 300])
@pytest.mark.parametrize("keys", [(40, 41), (0, 512)])
def test_keys_of_nan_reach_the_rows_that_see_them(new, splits, keys):
    """One key, and all keys of a split: NaN logits are not taken for keys that are not there."""
    x = _make([2048], [new], 2, 1, 2, 64, 16, 32, 19)
    j = torch.arange(*keys)
    x["kp"][x["table"][0].long()[j // 32], j % 32] = float("nan")
    out, l2 = _attend(x, splits)
    assert torch.isnan(out).all() and torch.isnan(l2).all()


@pytest.mark.parametrize("splits", [1, 4])
def test_keys_of_nan_are_not_seen_before_their_time(splits):
    """New tokens whose own key is NaN leave the tokens before them as they were."""
    for new in (5, 200):
        x = _make([700], [new], 4, 2, 4, 128, 32, 64, 23)
        ref, lse, _ = PO.attention(x, True)
        j = torch.tensor([700 - new // 2 - 1])  # new token `at`'s own key
        at = new - new // 2 - 1
        x["kp"][x["table"][0].long()[j // 64], j % 64] = float("nan")
        out, l2 = _attend(x, splits)
        _close_out("before", out[:at], ref[:at])
        _close_lse(l2[:, :at], lse[:, :at])
        assert torch.isnan(out[at:]).all() and torch.isnan(l2[:, at:]).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [8, 8, 8], [150, 70, 150]])
@pytest.mark.parametrize("bad", [-1, "past the pool", 1 << 30])
@pytest.mark.parametrize("page", [16, 128])
def test_page_ids_outside_the_pool_are_recorded(new, bad, page):
    """An entry within a sequence's length: recorded, its keys read as zeros, other sequences untouched."""
    from fna2_b200.paged import flash_naylis_paged, naylis_key_weights
    x = _make([500, 400, 300], new, 4, 2, 4, 64, 16, page, 29)
    at = 256 // page
    x["kp"][x["table"][1, at].long()] = 0.0
    x["vp"][x["table"][1, at].long()] = 0.0
    x["rp"][x["table"][1, at].long()] = 0.0
    ref, lse, w = PO.attention(x, True)
    d, pool = _dev(x), _pool(x)
    d["table"][1, at] = pool.num_pages if bad == "past the pool" else bad
    assert _status() == 0
    kw = dict(r_q=d["rq"], graph_scale=d["gs"])
    out, l2 = flash_naylis_paged(d["q"], pool, d["table"], d["lens"], d["cu"], max(new), return_lse=True, **kw)
    assert _status() == 641
    _close_out("out", out, ref)
    _close_lse(l2, lse)
    got = naylis_key_weights(d["q"], l2, pool, d["table"], d["lens"], d["cu"], max(new), **kw)
    assert _status() == 641
    _close_w(got, w)
