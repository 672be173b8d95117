"""GPU tests of the paged attention with many query heads per KV head, at the ranks where the
R_k tiles of a group are largest (tolerances as in test_gpu_paged)."""
import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_paged import _close_lse, _close_out, _close_w, _dev, _make, _pool, _status

pytestmark = pytest.mark.gpu

NEW = {"single": [1, 1, 1], "one": [1], "drafted": [3, 1, 2], "eight": [8, 0, 5], "mixed": [1, 90, 3]}


@pytest.mark.parametrize("group,kv_heads,graph,D,rank", [
    (13, 2, 26, 128, 32), (14, 1, 14, 128, 24), (16, 2, 32, 128, 32), (16, 1, 9, 128, 32), (23, 1, 23, 128, 32),
    (24, 2, 48, 128, 24), (25, 1, 25, 128, 32), (32, 1, 32, 128, 32), (64, 1, 64, 128, 32), (130, 1, 130, 128, 24),
    (16, 1, 16, 64, 32), (64, 1, 50, 64, 32)])
@pytest.mark.parametrize("kind", sorted(NEW))
def test_large_groups(group, kv_heads, graph, D, rank, kind):
    from fna2_b200.paged import flash_naylis_paged
    new = NEW[kind]
    lens = [333, 120, 64][:len(new)]
    x = _make(lens, new, group * kv_heads, kv_heads, graph, D, rank, 32, group + D)
    d = _dev(x)
    w = torch.zeros(len(lens), kv_heads, x["table"].shape[1] * 32, device="cuda")
    out, lse = flash_naylis_paged(d["q"], _pool(x), d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                                  graph_scale=d["gs"], return_lse=True, key_weights=w)
    ro, rl, rw = PO.attention(x, True)
    _close_out("out", out, ro)
    _close_lse(lse, rl)
    _close_w(w, rw)
    assert _status() == 0
