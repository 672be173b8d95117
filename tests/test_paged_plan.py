"""CPU tests of the choices of a paged attention call: every accepted shape has a kernel that
runs it, and the workspace stays within its bound.  The size query makes the choices that the
call makes, and refuses what the call refuses."""
import ctypes

import pytest

from fna2_b200 import _lib


def _query(G, kv_heads, D, rank, tokens, batch, max_k, weights=False, num_pages=1 << 12, page=64, total=None):
    buf = ctypes.create_string_buffer(1 << 10)
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    H = G * kv_heads
    kv = _lib.Fna2PagedKV(num_pages, page, kv_heads, H, D, rank, base, page * kv_heads * D, kv_heads * D, D, base,
                          page * kv_heads * D, kv_heads * D, D, base, page * H * rank, H * rank, rank)
    at = _lib.Fna2PagedAttnArgs(batch, H, tokens * batch if total is None else total, tokens, max_k, max_k // page, 1, 0,
                                0.088, base, max_k // page, base, base, base, H * D, D, base, H * rank, rank, base, base,
                                H * D, D, None, 0, base if weights else None, kv_heads * max_k, max_k, 0)
    lib = _lib.load()
    n = lib.fna2_paged_attn_workspace_size(kv, at)
    return n, lib.fna2_last_error().decode()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rank", [8, 16, 24, 32])
def test_every_group_size_has_a_kernel(D, rank):
    """1 to 64 query heads per KV head and more, one token to a chunk, alone and in batches."""
    for G in list(range(1, 65)) + [96, 128, 129, 200]:
        for tokens in list(range(1, 34)) + [300]:
            for batch in (1, 3):
                _, error = _query(G, 1, D, rank, tokens, batch, 4096)
                assert error == "", (G, tokens, batch, error)


@pytest.mark.parametrize("total,G,kv_heads,batch,tokens,max_k", [
    (26071, 16, 1, 16130, 31, 907776), (33172, 8, 1, 30805, 74, 137344), (1 << 21, 4, 2, 60000, 2000, 8192),
    (1 << 25, 1, 1, 65535, 1 << 20, 4096)])
def test_many_sequences_and_tokens_are_accepted(total, G, kv_heads, batch, tokens, max_k):
    """Splits of long keys times tens of thousands of short sequences: the grid has room for them."""
    _, error = _query(G, kv_heads, 128, 16, tokens, batch, max_k, total=total)
    assert error == ""


@pytest.mark.parametrize("batch,tokens,group", [(256, 1, 4), (64, 8, 4), (64, 8, 1), (64, 1, 32), (2000, 1, 4)])
@pytest.mark.parametrize("pages", [1 << 12, 1 << 14])
def test_workspace_of_key_weights_is_bounded(batch, tokens, group, pages):
    """Bounds of 131,072 keys, which one sequence of a batch may reach: never more than half of the pool's K
    (256 MB at least) and 2 GB, beside what a call without weights takes."""
    plain, _ = _query(group, 8, 128, 16, tokens, batch, 131072, num_pages=pages)
    n, error = _query(group, 8, 128, 16, tokens, batch, 131072, weights=True, num_pages=pages)
    k_bytes = pages * 64 * 8 * 128 * 2
    tokens_bytes = batch * tokens * 8 * group * (4 + 2 * (2 * 16 + 16)) + 4096  # LSE, R~_q and LSE columns
    assert error == "" and n - plain <= max(256e6, min(2e9, k_bytes / 2)) + tokens_bytes


def test_workspace_keeps_the_logits_of_ordinary_calls():
    """A pool filled by equal sequences: what their logits take is within the limit."""
    plain, _ = _query(4, 8, 128, 16, 1, 64, 4096, num_pages=64 * 64)
    n, _ = _query(4, 8, 128, 16, 1, 64, 4096, weights=True, num_pages=64 * 64)
    assert n - plain >= 64 * 32 * 4096 * 4
