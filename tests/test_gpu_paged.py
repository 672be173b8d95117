"""GPU tests of the paged-cache operators (append, attention, key weights,
eviction) against plain implementations in 64 bits.

Tolerances, from the arithmetic: outputs are bf16 (one rounding, at most 2^-9 of
the value) of sums whose probabilities were rounded to bf16 (2^-9 each, averaging
out), so 2^-8 of the value plus 2^-8 of the largest value covers both.  LSE and
key weights are fp32: logits carry the bias to 2^-17 of it and fp32 accumulation
noise, |S| stays below about 30 here, so 30 * 2^-17 + 1e-5 absolute on the LSE and,
since w = exp(S - LSE), relative 5e-4 on the weights bound them (typical errors
are two orders smaller; the second bound below, in the 2-norm, is 2e-5)."""
import math

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu


def _make(lens, new, H, H_KV, H_G, D, R, page, seed, layout="token", garbage=True, heads_scale=1.0):
    """A pool with the sequences' pages scattered over it, NaN in every slot that no key uses."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    pages = [-(-n // page) for n in lens]
    P = sum(pages) + 2
    order = torch.randperm(P, generator=g).int()
    maxp = max(1, max(pages))
    table = torch.full((B, maxp), -1, dtype=torch.int32)
    fill = float("nan") if garbage else 0.0
    kp = torch.full((P, page, H_KV, D), fill).bfloat16()
    vp = kp.clone()
    rp = torch.full((P, page, H_G, R), fill).bfloat16() if H_G else None
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
        j = torch.arange(lens[b])
        where = (table[b].long()[j // page], j % page)
        kp[where] = torch.randn(lens[b], H_KV, D, generator=g).bfloat16()
        vp[where] = torch.randn(lens[b], H_KV, D, generator=g).bfloat16()
        if H_G:
            rp[where] = (torch.randn(lens[b], H_G, R, generator=g) * R ** -0.5).bfloat16()
    T = sum(new)
    q = (torch.randn(T, H, D, generator=g) * heads_scale).bfloat16()
    rq = (torch.randn(T, H_G, R, generator=g) * R ** -0.5).bfloat16() if H_G else None
    gs = torch.randn(H_G, generator=g) if H_G else None
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    return dict(kp=kp, vp=vp, rp=rp, table=table, lens=lens, cu=cu, q=q, rq=rq, gs=gs, new=new)


def _pool(x, layout="token"):
    from fna2_b200.paged import PagedKV

    def put(t):
        if t is None:
            return None
        if layout == "head":  # [P, H, page, X] storage
            return t.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        return t.cuda()
    return PagedKV(put(x["kp"]), put(x["vp"]), put(x["rp"]))


def _dev(x):
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    return dict(q=c(x["q"]), table=c(x["table"]), lens=torch.tensor(x["lens"], dtype=torch.int32, device="cuda"),
                cu=c(x["cu"]), rq=c(x["rq"]), gs=c(x["gs"]))


def _close_out(name, got, ref):
    got, ref = got.float().cpu().double(), ref.cpu()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    bound = 2.0 ** -8 * (ref.abs() + ref.abs().max())
    assert ((got - ref).abs() <= bound).all(), f"{name}: {((got - ref).abs() / bound).max():.3g} of the bound"


def _close_lse(got, ref):
    got, ref = got.cpu().double(), ref.cpu()
    none = torch.isinf(ref)
    assert torch.equal(none, torch.isinf(got)) and (got[none] < 0).all()
    assert ((got - ref)[~none].abs() <= 30 * 2.0 ** -17 + 1e-5).all()


def _close_w(got, ref, base=None):
    """base: what the weights were added to (one fp32 rounding of each sum)."""
    got, ref = got.cpu().double(), ref.cpu()
    more = torch.zeros_like(ref) if base is None else 2.0 ** -23 * (base.double() + ref)
    ref0, ref = ref, ref if base is None else ref + base.double()
    assert ((got - ref).abs() <= 5e-4 * ref0 + 1e-9 + more).all()
    assert (got - ref).norm() <= 2e-5 * ref0.norm() + 1e-9 + more.norm()


def _status():
    from fna2_b200 import _lib
    torch.cuda.synchronize()
    return _lib.load().fna2_device_status(1)


CASES = [
    # lens (cached keys, the new ones' included), new, H, H_KV, H_G, D, R, page
    ([1], [1], 4, 4, 4, 64, 8, 16),
    ([257, 1, 64, 0, 129], [1, 1, 1, 0, 1], 8, 2, 8, 128, 16, 16),
    ([300, 17, 1000], [1, 1, 1], 6, 3, 0, 64, 16, 64),
    ([515, 40], [1, 1], 24, 1, 24, 128, 16, 32),
    ([700, 33, 64], [5, 3, 7], 8, 2, 5, 128, 24, 32),
    ([500, 130], [16, 9], 4, 4, 4, 64, 32, 128),
    ([130, 300, 5, 1], [130, 100, 5, 1], 4, 2, 3, 128, 32, 64),
    ([1000, 2, 700], [300, 1, 513], 2, 2, 2, 64, 16, 16),
    ([600, 77, 1500], [1, 1, 1], 16, 2, 16, 128, 32, 64),  # wide rows of few tokens
    ([600, 77, 1500], [1, 2, 2], 16, 2, 13, 128, 24, 64),
    ([3, 10], [7, 12], 4, 2, 4, 64, 16, 16),  # fewer cached keys than new tokens: the first rows see none
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_and_weights(case, causal):
    from fna2_b200.paged import flash_naylis_paged, naylis_key_weights
    lens, new, H, H_KV, H_G, D, R, page = case
    x = _make(lens, new, H, H_KV, H_G, D, R, page, 11 + H + D + len(lens))
    d = _dev(x)
    pool = _pool(x)
    w0 = torch.rand(len(lens), H_KV, x["table"].shape[1] * page)
    w = w0.cuda()
    out, lse = flash_naylis_paged(d["q"], pool, d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                                  graph_scale=d["gs"], is_causal=causal, return_lse=True)
    ro, rl, rw = PO.attention(x, causal)
    _close_out("out", out, ro)
    _close_lse(lse, rl)
    out2 = flash_naylis_paged(d["q"], pool, d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                              graph_scale=d["gs"], is_causal=causal, key_weights=w, max_seqlen_k=max(lens))
    _close_out("out with weights", out2, ro)
    _close_w(w, rw, w0)
    w2 = naylis_key_weights(d["q"], lse, pool, d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                            graph_scale=d["gs"], is_causal=causal)
    _close_w(w2, rw)
    assert _status() == 0


@pytest.mark.parametrize("splits", [1, 2, 7])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 200]])
def test_forced_splits(splits, new):
    from fna2_b200.paged import flash_naylis_paged
    lens = [900, 33, 2048]
    x = _make(lens, new, 8, 4, 8, 128, 16, 64, 3)
    d = _dev(x)
    w = torch.zeros(3, 4, x["table"].shape[1] * 64, device="cuda")
    out, lse = flash_naylis_paged(d["q"], _pool(x), d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                                  graph_scale=d["gs"], return_lse=True, num_splits=splits, key_weights=w)
    ro, rl, rw = PO.attention(x, True)
    _close_out("out", out, ro)
    _close_lse(lse, rl)
    _close_w(w, rw)


@pytest.mark.parametrize("new", [[1, 1], [5, 2], [140, 200]])
def test_strides_and_layouts(new):
    """Head-major pool storage, q and r_q as slices of wider tensors, a page table that is a slice."""
    from fna2_b200.paged import flash_naylis_paged
    lens = [333, 250]
    x = _make(lens, new, 4, 2, 4, 128, 16, 32, 8)
    d = _dev(x)
    T = sum(new)
    wide = torch.randn(T, 6, 256, device="cuda").bfloat16()
    wide[:, 1:5, 64:192] = d["q"]
    rwide = torch.randn(T, 5, 32, device="cuda").bfloat16()
    rwide[:, 1:, 8:24] = d["rq"]
    twide = torch.full((2, 40), -7, dtype=torch.int32, device="cuda")
    twide[:, 3:3 + d["table"].shape[1]] = d["table"]
    out, lse = flash_naylis_paged(wide[:, 1:5, 64:192], _pool(x, "head"), twide[:, 3:3 + d["table"].shape[1]],
                                  d["lens"], d["cu"], max(new), r_q=rwide[:, 1:, 8:24], graph_scale=d["gs"],
                                  return_lse=True)
    ro, rl, _ = PO.attention(x, True)
    _close_out("out", out, ro)
    _close_lse(lse, rl)


@pytest.mark.parametrize("new", [[1] * 150, [2] * 131 + [40] * 3])
def test_many_sequences(new):
    """More sequences than a CTA looks through at once, lengths from 0 on; one of many more keys than the rest."""
    from fna2_b200.paged import flash_naylis_paged, naylis_key_weights
    lens = [b * 7 % 90 for b in range(len(new))]
    lens[77] = 5000
    x = _make(lens, new, 2, 1, 2, 64, 16, 16, 3)
    d, pool = _dev(x), _pool(x)
    out, lse = flash_naylis_paged(d["q"], pool, d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                                  graph_scale=d["gs"], return_lse=True)
    ro, rl, rw = PO.attention(x, True)
    _close_out("out", out, ro)
    _close_lse(lse, rl)
    _close_w(naylis_key_weights(d["q"], lse, pool, d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                                graph_scale=d["gs"]), rw)
    assert _status() == 0


@pytest.mark.parametrize("T", [0, 3, 200])
def test_key_weights_start_from_zero(T):
    """Fresh weights: also those of keys past a sequence's end, and without a query."""
    from fna2_b200.paged import naylis_key_weights
    x = _make([300, 40], [T, 0], 4, 2, 4, 64, 16, 32, 5)
    d, pool = _dev(x), _pool(x)
    lse = torch.zeros(4, T, device="cuda")
    shape = (2, 2, x["table"].shape[1] * 32)
    dirty = [torch.full(shape, float("nan"), device="cuda") for _ in range(4)]
    del dirty  # their memory is handed out again
    w = naylis_key_weights(d["q"], lse, pool, d["table"], d["lens"], d["cu"], T, r_q=d["rq"], graph_scale=d["gs"])
    w2 = naylis_key_weights(d["q"], lse, pool, d["table"], d["lens"], d["cu"], T, r_q=d["rq"], graph_scale=d["gs"],
                            key_weights=torch.zeros(shape, device="cuda"))
    assert torch.equal(w, w2) and (w[1] == 0).all() and (w[0, :, 300:] == 0).all() and (T == 0 or (w[0] > 0).any())
    assert _status() == 0


def test_rows_equal_prefill_and_chunks_agree():
    """A prompt attended in chunks over the pages equals the packed prefill op, row for row."""
    from fna2_b200 import flash_naylis_attn
    from fna2_b200.paged import flash_naylis_paged
    L, H, H_KV, D, R = 700, 4, 2, 128, 32
    x = _make([L], [L], H, H_KV, H, D, R, 64, 21)
    d, pool = _dev(x), _pool(x)
    j = torch.arange(L)
    at = (x["table"][0].long()[j // 64], j % 64)
    k, v, rk = (x[n][at].cuda() for n in ("kp", "vp", "rp"))
    cu = torch.tensor([0, L], dtype=torch.int32, device="cuda")
    ref = flash_naylis_attn(d["q"], k, v, d["rq"], rk, d["gs"], is_causal=True, cu_seqlens_q=cu, cu_seqlens_k=cu,
                            max_seqlen_q=L, max_seqlen_k=L).float()
    a = 0
    for n in (1, 255, 3, 400, 41):
        e = a + n
        o = flash_naylis_paged(d["q"][a:e], pool, d["table"], torch.tensor([e], dtype=torch.int32, device="cuda"),
                               torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, r_q=d["rq"][a:e],
                               graph_scale=d["gs"]).float()
        # two kernels that each meet the bound of this file against 64 bits (the prefill one rounds the bias once more)
        assert ((o - ref[a:e]).abs() <= 2.0 ** -6 * (ref[a:e].abs() + ref.abs().max())).all()
        a = e


@pytest.mark.parametrize("new", [[1], [3], [130]])
def test_extreme_logits(new):
    """Large logits of both signs: the running maximum keeps every exponent in range."""
    from fna2_b200.paged import flash_naylis_paged
    x = _make([600], new, 2, 1, 2, 64, 16, 32, 5, heads_scale=60.0)
    d = _dev(x)
    out, lse = flash_naylis_paged(d["q"], _pool(x), d["table"], d["lens"], d["cu"], max(new), r_q=d["rq"],
                                  graph_scale=d["gs"], return_lse=True)
    ro, rl, _ = PO.attention(x, True)
    # |S| up to 300: fp32 logits are good to 300 * 2^-22 or so, P to that absolute error
    _close_out("out", out, ro)
    assert ((lse.cpu().double() - rl).abs() <= 2e-3).all()


def test_other_stream_and_repeat():
    """Work goes to the current stream, and two runs agree bit for bit."""
    from fna2_b200.paged import flash_naylis_paged
    x = _make([900, 500], [1, 120], 4, 4, 4, 128, 16, 64, 9)
    d, pool = _dev(x), _pool(x)

    def run():
        w = torch.zeros(2, 4, x["table"].shape[1] * 64, device="cuda")
        o, l = flash_naylis_paged(d["q"], pool, d["table"], d["lens"], d["cu"], 120, r_q=d["rq"], graph_scale=d["gs"],
                                  return_lse=True, key_weights=w)
        return o, l, w
    first = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = run()
    s.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_back_to_back_and_captured_calls():
    """Operators that follow each other without a pause, directly and from a captured graph: each one's
    results, read by the next, are complete (bit for bit the results of calls with pauses between them)."""
    from fna2_b200.paged import flash_naylis_paged, naylis_evict, naylis_key_weights, qk_norm_rope_append
    new, lens = [1, 120, 3], [900, 500, 64]
    x = _make(lens, new, 4, 2, 4, 128, 16, 64, 9)
    d = _dev(x)
    T, before = sum(new), torch.tensor([a - b for a, b in zip(lens, new)], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(T, 2, 128, generator=g).bfloat16().cuda() for _ in range(2))
    rk = torch.randn(T, 4, 16, generator=g).bfloat16().cuda()
    extra = 3 * 2  # pages of the compacted sequences
    for n in ("kp", "vp", "rp"):
        x[n] = torch.cat([x[n].nan_to_num(0.0), torch.zeros(extra, *x[n].shape[1:]).bfloat16()])
    tout = (torch.arange(extra, dtype=torch.int32) + x["kp"].shape[0] - extra).reshape(3, 2).cuda()

    def chain(pool, pause):
        wait = torch.cuda.synchronize if pause else lambda: None
        q = qk_norm_rope_append(d["q"], k, v, pool, d["table"], before, d["cu"], r_k=rk)
        wait()
        w = torch.zeros(3, 2, x["table"].shape[1] * 64, device="cuda")
        out, lse = flash_naylis_paged(q, pool, d["table"], d["lens"], d["cu"], 120, r_q=d["rq"], graph_scale=d["gs"],
                                      return_lse=True, key_weights=w)
        wait()
        w2 = naylis_key_weights(q, lse, pool, d["table"], d["lens"], d["cu"], 120, r_q=d["rq"], graph_scale=d["gs"])
        wait()
        kept, n, wo = naylis_evict(w2, pool, d["table"], d["lens"], 100, tout, recent=8, sink=2, heads=4)
        wait()
        one = torch.arange(4, dtype=torch.int32, device="cuda")
        last = flash_naylis_paged(q[:3], pool, tout, n, one, 1, r_q=d["rq"][:3], graph_scale=d["gs"])
        return q, out, lse, w, w2, kept, n, wo, last
    want = chain(_pool(x), True)
    fresh = _pool(x)
    torch.cuda.synchronize()
    got = chain(fresh, False)
    pool = _pool(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain(pool, False)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, captured):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert _status() == 0


def test_bad_lengths_are_skipped_and_recorded():
    from fna2_b200.paged import flash_naylis_paged, naylis_evict, naylis_key_weights
    x = _make([300, 200, 100], [1, 1, 1], 4, 4, 4, 64, 16, 32, 2)
    d, pool = _dev(x), _pool(x)
    ref, _, _ = PO.attention(x, True)
    assert _status() == 0
    for bad in (-5, 10 ** 6):
        lens = d["lens"].clone()
        lens[1] = bad
        out, lse = flash_naylis_paged(d["q"], pool, d["table"], lens, d["cu"], 1, r_q=d["rq"], graph_scale=d["gs"],
                                      return_lse=True)
        assert _status() == 641
        _close_out("others", out[[0, 2]], ref[[0, 2]])
        w = naylis_key_weights(d["q"], torch.zeros_like(lse), pool, d["table"], lens, d["cu"], 1, r_q=d["rq"],
                               graph_scale=d["gs"])
        assert _status() == 641 and (w[1] == 0).all()
        tout = torch.zeros(3, 1, dtype=torch.int32, device="cuda") + pool.num_pages - 1
        kept, n, _ = naylis_evict(w, pool, d["table"], lens, 8, tout, heads=4)
        assert _status() == 651 and n.tolist() == [8, 0, 8] and (kept[1] == -1).all()


EVICT = [
    # lens, H, H_KV, H_G, D, R, page, budget, recent, sink
    ([600, 512, 100, 0, 513], 4, 4, 4, 64, 8, 16, 512, 64, 4),
    ([1000, 2500], 8, 2, 5, 128, 16, 64, 300, 0, 0),
    ([70], 2, 1, 0, 128, 16, 32, 64, 64, 0),   # only the newest
    ([40, 41], 2, 2, 2, 64, 32, 16, 1, 0, 1),  # only the first
    ([5000], 3, 3, 3, 64, 24, 128, 4999, 10, 3),
    ([50000, 7], 1, 1, 1, 64, 8, 128, 1000, 100, 4),  # weights that do not fit in shared memory
    ([49500], 2, 1, 1, 64, 8, 128, 500, 10, 0),
]


@pytest.mark.parametrize("case", EVICT)
@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_evict(case, kind):
    from fna2_b200.paged import naylis_evict
    lens, H, H_KV, H_G, D, R, page, budget, recent, sink = case
    x = _make(lens, [1] * len(lens), H, H_KV, H_G, D, R, page, 4 + budget)
    d = _dev(x)
    g = torch.Generator().manual_seed(budget)
    B, cap = len(lens), x["table"].shape[1] * page
    w = torch.rand(B, H_KV, cap, generator=g) * 10
    if kind == "ties":
        w = torch.floor(w)
    elif kind == "special":
        r = torch.rand(w.shape, generator=g)
        for v, lo, hi in ((0.0, 0, .2), (-0.0, .2, .4), (float("inf"), .4, .5), (float("-inf"), .5, .55),
                          (float("nan"), .55, .6), (1e-42, .6, .7), (-3.0, .7, .8)):
            w[(r >= lo) & (r < hi)] = v
    out_pages = -(-budget // page)
    base = x["kp"].shape[0]
    total = base + B * out_pages
    pools = {}
    for n in ("kp", "vp", "rp"):
        if x[n] is not None:
            big = torch.zeros(total, *x[n].shape[1:]).bfloat16()
            big[:base] = x[n]
            pools[n] = big.cuda()
    from fna2_b200.paged import PagedKV
    pool = PagedKV(pools["kp"], pools["vp"], pools.get("rp"))
    perm = torch.randperm(B * out_pages, generator=g).int() + base
    tout = perm.reshape(B, out_pages)
    kept, n_out, w_out = naylis_evict(w.cuda(), pool, d["table"], d["lens"], budget, tout.cuda(), recent=recent,
                                      sink=sink, heads=H, max_seqlen_k=max(lens))
    assert _status() == 0
    ref = PO.evict(w, lens, budget, recent, sink)
    assert n_out.tolist() == [min(n, budget) for n in lens]
    kept, w_out = kept.cpu(), w_out.cpu()
    for b in range(B):
        n = min(lens[b], budget)
        dst = torch.arange(n)
        to = (tout[b].long()[dst // page], dst % page)
        for h in range(H_KV):
            assert kept[b, h].tolist() == ref[b][h] + [-1] * (budget - n)
            src = torch.tensor(ref[b][h], dtype=torch.long)
            assert torch.equal(w_out[b, h, :n].nan_to_num(7.5), w[b, h, src].nan_to_num(7.5))
            assert (w_out[b, h, n:] == 0).all()
            frm = (x["table"][b].long()[src // page], src % page)
            for name in ("kp", "vp"):
                assert torch.equal(pools[name][to[0], to[1], h].cpu(), x[name][frm[0], frm[1], h])
            for hh in range(h * (H // H_KV), min(H_G, (h + 1) * (H // H_KV))):
                assert torch.equal(pools["rp"][to[0], to[1], hh].cpu(), x["rp"][frm[0], frm[1], hh])
    for name in pools:  # the old pages stay as they were
        assert torch.equal(pools[name][:base].cpu().view(torch.int16), x[name].view(torch.int16))


class _Mod:
    def __init__(self, **kw):
        self.__dict__.update(kw)


@pytest.mark.parametrize("H,H_KV,H_G,D,R", [(4, 4, 4, 64, 8), (24, 3, 10, 128, 32), (2, 1, 0, 128, 16)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("mode", ["both", "norm", "rope", "none"])
def test_append(H, H_KV, H_G, D, R, dtype, wdtype, mode):
    """Rows equal the packed training transform bit for bit at the same positions, the pages
    hold them, and nothing else in the pool changes."""
    from fna2_b200.paged import PagedKV, qk_norm_rope_append
    from fna2_b200.qk_prep import apply_qk_norm_rope_varlen
    g = torch.Generator().manual_seed(H + D)
    past, new, page = [0, 31, 16, 5, 70], [1, 40, 0, 16, 3], 16
    B, T, lead = 5, 60, 2  # two tokens outside every sequence on either side
    x = _make([a + b for a, b in zip(past, new)], new, H, H_KV, H_G, D, R, page, 77, garbage=False)
    before = {n: x[n].clone() for n in ("kp", "vp", "rp") if x[n] is not None}
    pool = PagedKV(*(None if x[n] is None else x[n].cuda() for n in ("kp", "vp", "rp")))
    Tt = T + 2 * lead
    q, k, v = (torch.randn(Tt, h, D, generator=g).to(dtype).cuda() for h in (H, H_KV, H_KV))
    rk = torch.randn(Tt, H_G, R, generator=g).to(dtype).cuda() if H_G else None
    norms = (None, None)
    if mode in ("both", "norm"):
        norms = tuple(_Mod(weight=(1 + 0.2 * torch.randn(D, generator=g)).to(wdtype).cuda(), eps=1e-6)
                      for _ in range(2))
    inv = 10000.0 ** (-torch.arange(0, D, 2).float() / D)
    rope = _Mod(inv_freq=inv.cuda()) if mode in ("both", "rope") else None
    cu = (torch.tensor([0] + list(torch.tensor(new).cumsum(0))) + lead).int().cuda()
    lens = torch.tensor(past, dtype=torch.int32, device="cuda")
    pos = torch.tensor([a + 9 for a in past], dtype=torch.int32, device="cuda")
    qo = qk_norm_rope_append(q, k, v, pool, x["table"].cuda(), lens, cu, r_k=rk, positions=pos, q_norm=norms[0],
                             k_norm=norms[1], rope=rope)
    assert _status() == 0
    want = {n: t.clone() for n, t in before.items()}
    c = cu.tolist()
    for b in range(B):
        n, p0 = new[b], past[b] + 9
        if n == 0:
            continue
        # the training transform on a sequence long enough to hold these positions, rows at its end
        pad = lambda t: torch.cat([torch.zeros(p0, *t.shape[1:], dtype=t.dtype, device="cuda"), t[c[b]:c[b + 1]]])  # noqa: E731,B023
        cb = torch.tensor([0, p0 + n], dtype=torch.int32, device="cuda")
        rq_, rk_ = apply_qk_norm_rope_varlen(pad(q), pad(k), cb, norms[0], norms[1], rope)
        assert torch.equal(qo[c[b]:c[b + 1]], rq_[p0:])
        j = torch.arange(past[b], past[b] + n)
        at = (x["table"][b].long()[j // page], j % page)
        want["kp"][at] = rk_[p0:].cpu()
        want["vp"][at] = v[c[b]:c[b + 1]].bfloat16().cpu()
        if H_G:
            want["rp"][at] = rk[c[b]:c[b + 1]].bfloat16().cpu()
        if dtype == torch.float32 or wdtype == torch.float32 and mode != "rope":
            # against 64 bits: one bf16 rounding, plus fp32 angles below 100 (2^-17 absolute)
            ref = PO.norm_rope(q[c[b]:c[b + 1]].cpu(), None if norms[0] is None else norms[0].weight.cpu(), 1e-6,
                               None if rope is None else inv, torch.arange(p0, p0 + n))
            assert ((qo[c[b]:c[b + 1]].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -14).all()
    for n, t in want.items():
        assert torch.equal({"kp": pool.k_pages, "vp": pool.v_pages, "rp": pool.rk_pages}[n].cpu(), t)


def test_append_skips_what_does_not_fit():
    from fna2_b200.paged import qk_norm_rope_append
    x = _make([64, 40], [1, 1], 2, 2, 2, 64, 16, 32, 6, garbage=False)
    pool, table = _pool(x), x["table"].cuda()
    t = lambda h, d: torch.ones(2, h, d, device="cuda").bfloat16()  # noqa: E731
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for lens, bad_table in (([64, 40], False), ([-1, 40], False), ([63, 40], True)):  # full, negative, page outside
        tab = table.clone()
        if bad_table:
            tab[0, 1] = pool.num_pages
        k0 = pool.k_pages.clone()
        qk_norm_rope_append(t(2, 64), t(2, 64), t(2, 64), pool, tab,
                            torch.tensor(lens, dtype=torch.int32, device="cuda"), cu, r_k=t(2, 16))
        assert _status() == 631
        changed = (pool.k_pages != k0).flatten(2).any(-1).nonzero().tolist()
        assert changed in ([], [[int(table[1, 1]), 8]])  # the other sequence's slot 40
        pool.k_pages.copy_(k0)


def test_python_refusals():
    from fna2_b200.paged import PagedKV, flash_naylis_paged, naylis_evict, naylis_key_weights, qk_norm_rope_append
    x = _make([64, 40], [1, 1], 4, 2, 4, 64, 16, 32, 6)
    d, pool = _dev(x), _pool(x)
    ok = dict(q=d["q"], pool=pool, page_table=d["table"], cache_seqlens=d["lens"], cu_seqlens_q=d["cu"],
              max_seqlen_q=1, r_q=d["rq"], graph_scale=d["gs"])
    flash_naylis_paged(**ok)
    for name, value, kind in (("q", d["q"].float(), TypeError), ("q", d["q"][:, :, :32], ValueError),
                              ("r_q", None, ValueError), ("r_q", d["rq"][:1], ValueError),
                              ("cache_seqlens", d["lens"].long(), ValueError), ("cu_seqlens_q", d["lens"], ValueError),
                              ("page_table", d["table"][0], ValueError), ("graph_scale", d["gs"][:2], ValueError),
                              ("softmax_scale", -1.0, RuntimeError)):
        with pytest.raises(kind):
            flash_naylis_paged(**{**ok, name: value})
    with pytest.raises(ValueError, match="key_weights"):
        flash_naylis_paged(**ok, key_weights=torch.zeros(2, 2, 10, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        naylis_key_weights(lse=torch.zeros(4, 3, device="cuda"), **ok)
    w = torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="budget"):
        naylis_evict(w, pool, d["table"], d["lens"], 8, d["table"][:, :1], recent=9, heads=4)
    with pytest.raises(ValueError, match="page_table_out"):
        naylis_evict(w, pool, d["table"], d["lens"], 8, d["table"][:1], heads=4)
    with pytest.raises(TypeError, match="k must be"):
        qk_norm_rope_append(d["q"], d["q"][:, :2].float(), d["q"][:, :2], pool, d["table"], d["lens"], d["cu"])
    with pytest.raises(ValueError, match="r_k"):
        qk_norm_rope_append(d["q"], d["q"][:, :2], d["q"][:, :2], pool, d["table"], d["lens"], d["cu"])
    with pytest.raises(ValueError, match="shape of k_pages"):
        PagedKV(pool.k_pages, pool.v_pages[:, :, :1])
    assert _status() == 0
