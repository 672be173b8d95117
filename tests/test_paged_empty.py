"""CPU tests: an empty batch is no error in any of the paged-cache operators (its tensors hold no
element, so their pointers may be NULL), and with a sequence in it the same pointers are."""
import pytest

from fna2_b200 import _lib
from test_paged_refusals import args  # noqa: F401  (the fixture)


def _null(a, *fields):
    for f in fields:
        setattr(a, f, None)


def _calls(args):
    kv, at, ap, ev, _ = args
    lib = _lib.load()
    at.total_q = ap.total_tokens = 0
    _null(at, "page_table", "cache_seqlens", "q", "r_q", "out")
    _null(ap, "page_table", "cache_seqlens")
    _null(ev, "page_table", "page_table_out", "cache_seqlens", "key_weights", "kept", "seqlens_out", "weights_out")
    return {"attention": (at, lambda: lib.fna2_paged_attn(kv, at, None, 0, None)),
            "weights": (at, lambda: lib.fna2_key_weights(kv, at, None, 0, None)),
            "append": (ap, lambda: lib.fna2_paged_append(kv, ap, None)),
            "evict": (ev, lambda: lib.fna2_evict(kv, ev, None))}


@pytest.mark.parametrize("name", ["attention", "weights", "append", "evict"])
def test_empty_batch(args, name):  # noqa: F811
    a, call = _calls(args)[name]
    a.batch = 0
    assert call() == _lib.FNA2_OK, _lib.load().fna2_last_error().decode()
    a.batch = 1
    assert call() == _lib.FNA2_ERR_INVALID


def test_no_pages_no_keys(args):  # noqa: F811
    """Sequences that own no page have an empty table; their weights are empty as well."""
    kv, at, _, _, _ = args
    at.total_q, at.max_pages, at.max_seqlen_k, at.table_stride = 0, 0, 0, 1
    _null(at, "page_table", "q", "r_q", "out")
    lib = _lib.load()
    assert lib.fna2_paged_attn(kv, at, None, 0, None) == _lib.FNA2_OK
    assert lib.fna2_key_weights(kv, at, None, 0, None) == _lib.FNA2_OK
