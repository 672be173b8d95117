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


def test_weights_of_one_long_sequence_among_many():
    """Key weights of single tokens where their logits would take more than the pool: formed again."""
    from fna2_b200.paged import flash_naylis_paged
    lens = [3] * 300 + [70000] + [1] * 99
    x = _make(lens, [1] * 400, 8, 2, 8, 64, 8, 256, 40)
    d = _dev(x)
    w = torch.zeros(400, 2, x["table"].shape[1] * 256, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = flash_naylis_paged(d["q"], _pool(x), d["table"], d["lens"], d["cu"], 1, r_q=d["rq"], graph_scale=d["gs"],
                                  return_lse=True, key_weights=w, max_seqlen_k=70000)
    assert torch.cuda.max_memory_allocated() - before < 400e6  # the logits alone: 400 * 8 * 70,000 * 4 bytes = 900 MB
    ro, rl, rw = PO.attention(x, True)
    _close_out("out", out, ro)
    _close_lse(lse, rl)
    _close_w(w, rw)
