"""CPU tests of the paged-cache operators: the argument structs match the C layout, the C
entry points refuse bad arguments on the host (validation precedes any CUDA call), and the
Python layer refuses what it documents."""
import ctypes
import os
import subprocess

import pytest
import torch

from fna2_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_c(tmp_path):
    structs = {"Fna2PagedKV": ("rk_head_stride", "k"), "Fna2AppendArgs": ("inv_freq", "q_out"),
               "Fna2PagedAttnArgs": ("kw_head_stride", "lse"), "Fna2EvictArgs": ("weights_out", "key_weights")}
    src = tmp_path / "p.c"
    body = "".join(f'printf("%zu %zu %zu\\n", sizeof({s}), offsetof({s}, {f[0]}), offsetof({s}, {f[1]}));'
                   for s, f in structs.items())
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fna2.h"\nint main(){' + body + "}\n")
    exe = tmp_path / "p"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    want = []
    for s, f in structs.items():
        c = getattr(_lib, s)
        want += [ctypes.sizeof(c)] + [getattr(c, n).offset for n in f]
    assert got == want
    from fna2_b200 import paged  # the packed blocks of the Python layer end where the structures do
    for block, s in ((paged._ATTN_ARGS, _lib.Fna2PagedAttnArgs), (paged._APPEND_ARGS, _lib.Fna2AppendArgs),
                     (paged._EVICT_ARGS, _lib.Fna2EvictArgs)):
        assert block.size == ctypes.sizeof(s)


@pytest.fixture
def args():
    buf = ctypes.create_string_buffer(1 << 16)
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    kv = _lib.Fna2PagedKV(8, 64, 2, 4, 128, 16, base, 64 * 256, 256, 128, base, 64 * 256, 256, 128, base, 64 * 64, 64,
                          16)
    at = _lib.Fna2PagedAttnArgs(2, 4, 2, 1, 100, 2, 1, 0, 0.088, base, 2, base, base, base, 512, 128, base, 64, 16,
                                base, base, 512, 128, base, 2, None, 0, 0)
    row = lambda h, d: _lib.Fna2Rows(base, h * d, d)  # noqa: E731
    ap = _lib.Fna2AppendArgs(2, 4, 2, 1, 0, 1, 2, row(4, 128), row(2, 128), row(2, 128), row(4, 16), row(4, 128), base,
                             2, base, base, None, None, None, 1e-6, None)
    ev = _lib.Fna2EvictArgs(2, 4, 100, 2, 1, 64, 2, 8, base, 2, base, 1, base, base, 256, 128, base, base, base)
    return kv, at, ap, ev, buf


def _refused(rc, msg, code=_lib.FNA2_ERR_INVALID):
    assert rc == code
    assert msg in _lib.load().fna2_last_error().decode()


@pytest.mark.parametrize("field,value,msg", [
    ("head_dim", 96, "head_dim"), ("page_size", 48, "page_size"), ("page_size", 8, "page_size"),
    ("kv_heads", 3, "multiple of kv_heads"), ("rank", 12, "rank"), ("rank", 40, "rank"),
    ("graph_heads", 5, "graph_heads"), ("k", None, "null pool"), ("k_token_stride", 100, "strides"),
])
def test_pool_is_checked_by_every_entry(args, field, value, msg):
    kv, at, ap, ev, _ = args
    setattr(kv, field, value)
    lib = _lib.load()
    _refused(lib.fna2_paged_attn(kv, at, None, 0, None), msg)
    _refused(lib.fna2_key_weights(kv, at, None, 0, None), msg)
    _refused(lib.fna2_paged_append(kv, ap, None), msg)
    _refused(lib.fna2_evict(kv, ev, None), msg)
    assert lib.fna2_paged_attn_workspace_size(kv, at) == 0


@pytest.mark.parametrize("field,value,msg", [
    ("max_seqlen_k", 129, "max_seqlen_k"), ("softmax_scale", 0.0, "softmax_scale"), ("q", None, "null tensor"),
    ("q_head_stride", 100, "q must be"), ("r_q", None, "r_q"), ("cache_seqlens", None, "null sequence"),
    ("page_table", None, "page table"), ("batch", -1, "bad sizes"), ("table_stride", 1, "page table"),
])
def test_attention_refuses(args, field, value, msg):
    kv, at, _, _, _ = args
    setattr(at, field, value)
    _refused(_lib.load().fna2_paged_attn(kv, at, None, 0, None), msg)


def test_attention_workspace(args):
    kv, at, _, _, _ = args
    lib = _lib.load()
    at.num_splits = 2
    need = lib.fna2_paged_attn_workspace_size(kv, at)
    assert need > 0 and need % 256 == 0
    _refused(lib.fna2_paged_attn(kv, at, None, 0, None), "workspace", _lib.FNA2_ERR_WORKSPACE)
    _refused(lib.fna2_paged_attn(kv, at, at.q, need - 1, None), "workspace", _lib.FNA2_ERR_WORKSPACE)
    at.batch = 0
    assert lib.fna2_paged_attn(kv, at, None, 0, None) == _lib.FNA2_OK


def test_key_weights_refuse(args):
    kv, at, _, _, _ = args
    _refused(_lib.load().fna2_key_weights(kv, at, None, 0, None), "key_weights")


@pytest.mark.parametrize("clear,stride,offset,msg", [(96, 128, 0, "below max_seqlen_k"), (102, 128, 0, "multiple of 4"),
                                                      (128, 129, 0, "aligned"), (128, 128, 4, "aligned")])
def test_cleared_key_weights_refuse(args, clear, stride, offset, msg):
    kv, at, _, _, _ = args
    at.key_weights, at.kw_batch_stride, at.kw_head_stride, at.kw_clear = at.q + offset, 2 * stride, stride, clear
    _refused(_lib.load().fna2_key_weights(kv, at, None, 0, None), msg)


@pytest.mark.parametrize("field,value,msg", [
    ("in_dtype", 5, "in_dtype"), ("rope_dtype", 7, "rope_dtype"), ("eps", -1.0, "eps"),
    ("cu_seqlens", None, "null sequence"), ("total_tokens", -1, "bad sizes"), ("q_weight", 256, "both RMSNorm"),
])
def test_append_refuses(args, field, value, msg):
    kv, _, ap, _, _ = args
    setattr(ap, field, value)
    _refused(_lib.load().fna2_paged_append(kv, ap, None), msg)


def test_append_refuses_misaligned_rows(args):
    kv, _, ap, _, _ = args
    ap.v = _lib.Fna2Rows(ap.v.ptr + 2, 256, 128)
    _refused(_lib.load().fna2_paged_append(kv, ap, None), "aligned")


@pytest.mark.parametrize("field,value,msg", [
    ("budget", 0, "budget"), ("budget", 9, "budget"), ("budget", 65, "fewer than budget"), ("sink", -1, "sink"),
    ("max_seqlen_k", 200, "max_seqlen_k"), ("page_table_out", None, "output page table"), ("kept", None, "null"),
])
def test_evict_refuses(args, field, value, msg):
    kv, _, _, ev, _ = args
    setattr(ev, field, value)
    _refused(_lib.load().fna2_evict(kv, ev, None), msg)


def test_python_pool_refuses():
    from fna2_b200.paged import PagedKV
    k = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        PagedKV(k, k)
    with pytest.raises(TypeError, match="bfloat16"):
        PagedKV(k.float(), k)
