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
