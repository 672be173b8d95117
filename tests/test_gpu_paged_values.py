"""GPU tests of the paged attention with infinities and NaN among the values in use: they reach
the rows that the definition lets them reach, and no others, whichever kernel serves the row.

Tolerances are those of test_gpu_paged (their derivation is there)."""
import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_paged import _close_lse, _close_out, _dev, _make, _pool

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
