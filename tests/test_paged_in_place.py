"""CPU tests: a paged-cache call whose output is one of its inputs is refused (blocks that start later
would read what earlier ones have written)."""
import pytest

from fna2_b200 import _lib
from test_paged_refusals import _refused, args  # noqa: F401  (the fixture)


def test_attention_onto_its_queries(args):  # noqa: F811
    kv, at, _, _, _ = args
    at.num_splits, at.max_seqlen_q = 1, 1
    need = _lib.load().fna2_paged_attn_workspace_size(kv, at)
    assert need == 0 and at.out == at.q
    _refused(_lib.load().fna2_paged_attn(kv, at, None, 0, None), "must not be q")


@pytest.mark.parametrize("output,source", [("seqlens_out", "cache_seqlens"), ("weights_out", "key_weights")])
def test_eviction_onto_its_inputs(args, output, source):  # noqa: F811
    kv, _, _, ev, _ = args
    for i, name in enumerate(("seqlens_out", "weights_out")):
        setattr(ev, name, ev.cache_seqlens + 4096 * (i + 1))
    setattr(ev, output, getattr(ev, source))
    _refused(_lib.load().fna2_evict(kv, ev, None), output)
