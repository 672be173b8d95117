// Paged attention of sequences with many new tokens, on the tensor cores.
//
// Same definition as fna2_paged.cu.  The roles, the TMEM plan and the order of
// the MMAs are those of fna2_fwd_kernel (fna2_fwd.cu): one CTA per pair of
// 128-row query tiles of one query head, softmax warpgroups 0 / 1, a TMA warp and
// an MMA warp; S_i = Q_i K^T + R~_q,i R_k^T accumulates in TMEM, P goes back over
// it in bf16 and O_i += P_i V.  What differs:
//   - K, V and R_k tiles of 128 keys are gathered page by page: lane l of the TMA
//     warp looks up page l of the tile and issues its boxes (a box is at most a
//     page; its rows keep their place in the swizzled tile, whose pattern repeats
//     every 8 rows);
//   - R~_q is hi + lo (two K slices against the same R_k; see fna2_paged.cu), which
//     takes shared memory from V: V streams in half tiles of 64 keys, three of them
//     where rank > 16 and D = 128, else four;
//   - rows of V past a sequence's end hold whatever the page holds: the softmax
//     warps zero them before P V (P is 0 there, but 0 * NaN is not);
//   - a sequence's keys may be split over CTAs (`chunk` keys each) when there are
//     too few query tiles to fill the GPU; fna2_paged_many_join_kernel joins them.
// Bound: the hand-offs of the two query tiles' chains (product, TMEM load, exp2, TMEM store, product).
// 2,048 tokens over 30,717 keys, 32 heads, D = 128, rank 32: 1,440 us in a loop (830 TFLOP/s; SM clock
// 1,680 to 1,760 MHz under the power cap).  A key tile against both query tiles takes 5,200 to 5,600 clk,
// of which 2,560 are products and 2,048 exp2; with 148 equal CTAs the tensor pipe is active 52 % of the
// cycles, the exp2 pipe 42 %.
#include "fna2_paged.cuh"

namespace fna2 {

template <int D, int RP>
struct ManySmem {
  static constexpr int kQBytes = kBlockM * D * 2;
  static constexpr int kRBytes = kBlockM * RP * 2;  // R_q hi or lo of one query tile, R_k of one key tile
  static constexpr int kKBytes = kBlockN * D * 2;
  static constexpr int kVHalf = 64 * D * 2;         // 64 keys
  static constexpr int kVStages = (D == 128 && RP == 32) ? 3 : 4;
  static constexpr int kChunk = 128 * 128;  // 64 columns of a 128-row tile
  static constexpr int kVChunk = 64 * 128;  // 64 columns of a 64-row half tile
  static constexpr int oQ = 0;
  static constexpr int oRq = oQ + 2 * kQBytes;     // hi of tiles 0, 1
  static constexpr int oRqLo = oRq + 2 * kRBytes;  // lo of tiles 0, 1
  static constexpr int oK = oRqLo + 2 * kRBytes;   // 2 stages
  static constexpr int oRk = oK + 2 * kKBytes;     // 2 stages
  static constexpr int oV = oRk + 2 * kRBytes;     // kVStages half tiles
  static constexpr int oBar = oV + kVStages * kVHalf;
  static constexpr int kNumBars = 24;
  static constexpr int oMisc = oBar + kNumBars * 8;
  static constexpr int kUsed = oMisc + 16;
  static constexpr int kTotal = kUsed + 1024;
  static_assert(kTotal <= kMaxDynamicSmem, "shared memory budget");
  static_assert(kRBytes % 1024 == 0 && kVHalf % 1024 == 0, "swizzle atoms stay aligned");
};

enum ManyBar {
  kMbQFull = 0,
  kMbRqReady = 1,  // +tile
  kMbKFull = 3,    // +stage
  kMbKEmpty = 5,   // +stage
  kMbVFull = 7,    // +stage
  kMbVEmpty = 11,  // +stage
  kMbSFull = 15,   // +tile
  kMbPFull = 17,   // +tile
  kMbAllDone = 19,
};

struct ManyItem {
  PagedSeq sq;
  int b, pair, split, ns;
};

// Work item `idx` of the call: the sequences' (split, pair of query tiles), in
// packing order, the pairs of a split together (they read the same keys), heaviest first.  Every warp finds it by itself (a scan over
// the sequences, 32 a round); false when idx is past the last item.
__device__ __forceinline__ bool many_item(const PagedAttnParams& p, int idx, int lane, ManyItem* it) {
  int carry = 0;
  for (int base = 0; base < p.bd.B; base += 32) {
    const int b = base + lane;
    int cnt = 0, ns = 1;
    if (b < p.bd.B) {
      const PagedSeq s = paged_seq(p.bd, b);
      if (!s.ok) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
      if (s.n * p.G > p.few_rows) {
        ns = max(1, (s.len + p.chunk_many - 1) / p.chunk_many);
        cnt = (s.n + 2 * kBlockM - 1) / (2 * kBlockM) * ns;
      }
    }
    int incl = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, idx < carry + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int local = idx - carry - (__shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, cnt, src));
      it->b = base + src;
      it->ns = __shfl_sync(0xffffffffu, ns, src);
      it->sq = paged_seq(p.bd, it->b);
      const int pairs = (it->sq.n + 2 * kBlockM - 1) / (2 * kBlockM);
      it->split = local / pairs;
      it->pair = pairs - 1 - local % pairs;
      return true;
    }
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

template <int D, int RP>
__global__ void __launch_bounds__(kFwdThreads, 1)
    fna2_paged_many_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                           const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmRq,
                           const __grid_constant__ CUtensorMap tmRk, const PagedAttnParams p) {
  using L = ManySmem<D, RP>;
  constexpr int NV = L::kVStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::oMisc + 4);
  const int warp = warp_id(), lane = lane_id(), tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();

  ManyItem it;
  if (!many_item(p, blockIdx.x / p.H, lane, &it)) return;
  const PagedSeq sq = it.sq;
  const int h = blockIdx.x % p.H, hk = h / p.G;
  const bool graph = h < p.kv.hg;
  const int q0 = it.pair * 2 * kBlockM, past = sq.len - sq.n;
  // key tiles [t0, t1) of this split; n_t: how many of them each query tile sees
  const int t0 = it.split * (p.chunk_many / kBlockN);
  const int t1 = min(t0 + p.chunk_many / kBlockN, (sq.len + kBlockN - 1) / kBlockN);
  int n_t[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int qt = q0 + i * kBlockM;
    const int end = qt >= sq.n ? 0 : (p.causal ? past + min(sq.n, qt + kBlockM) : sq.len);
    n_t[i] = max(0, min((max(end, 0) + kBlockN - 1) / kBlockN, t1) - t0);
  }
  const int n_kv = max(n_t[0], n_t[1]);

  // Results of a row that sees no key of this split.
  auto write_none = [&](int q_local) {
    const int64_t tok = sq.q0 + q_local;
    if (it.ns == 1) {
      __nv_bfloat16* o = p.out + tok * p.o_st + h * p.o_sh;
      for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
      if (p.lse) p.lse[h * p.lse_sh + tok] = -INFINITY;
    } else {
      p.ws_ml[(tok * p.H + h) * p.ns + it.split] = make_float2(-INFINITY, 0.f);
    }
  };
  if (n_kv == 0) {
    if (tid < 2 * kBlockM && q0 + tid < sq.n) write_none(q0 + tid);
    return;
  }

  if (tid == 0) {
    mbar_init(&bars[kMbQFull], 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kMbRqReady + s], 4);
      mbar_init(&bars[kMbKFull + s], 1);
      mbar_init(&bars[kMbKEmpty + s], 1);
      mbar_init(&bars[kMbSFull + s], 1);
      mbar_init(&bars[kMbPFull + s], 4);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(&bars[kMbVFull + s], 1);
      mbar_init(&bars[kMbVEmpty + s], 1);
    }
    mbar_init(&bars[kMbAllDone], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 8) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      int q_bytes = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (n_t[i] > 0) q_bytes += L::kQBytes + (graph ? L::kRBytes : 0);
      mbar_expect_tx(&bars[kMbQFull], q_bytes);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (n_t[i] == 0) continue;
        const int qrow = sq.q0 + q0 + i * kBlockM;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + L::oQ + i * L::kQBytes + c * L::kChunk, &tmQ, &bars[kMbQFull], c * 64, qrow, h, 0);
        if (graph) tma_load_4d(smem + L::oRq + i * L::kRBytes, &tmRq, &bars[kMbQFull], 0, qrow, h, 0);
      }
    }
    __syncwarp();
    const int* table = p.kv.table + it.b * p.kv.table_sb;
    const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
    const int bk = min(1 << lg, kBlockN), bv = min(1 << lg, 64);  // rows of a K / V box
    // Lane l owns the l-th K box of a tile and the l-th V box of a half tile; boxes that start past
    // the sequence's end are not loaded.
    auto load_k = [&](int j) -> bool {
      const int s = j & 1, key = (t0 + j) * kBlockN + lane * bk;
      const bool mine = lane * bk < kBlockN && key < sq.len;
      const int page = mine ? __ldg(table + (key >> lg)) : 0;
      if (mine) check_page(p.kv, page);
      const bool free = j < 2 || mbar_wait(&bars[kMbKEmpty + s], ((j >> 1) - 1) & 1, abort_flag, 111);
      if (!__all_sync(0xffffffffu, free)) return false;
      const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_expect_tx(&bars[kMbKFull + s], boxes * bk * (D + (graph ? RP : 0)) * 2);
      __syncwarp();
      if (mine) {
        uint8_t* dk = smem + L::oK + s * L::kKBytes + lane * bk * 128;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(dk + c * L::kChunk, &tmK, &bars[kMbKFull + s], c * 64, key & mask, hk, page);
        if (graph)
          tma_load_4d(smem + L::oRk + s * L::kRBytes + lane * bk * RP * 2, &tmRk, &bars[kMbKFull + s], 0, key & mask,
                      h, page);
      }
      __syncwarp();
      return true;
    };
    auto load_v = [&](int hv) -> bool {  // half tile hv of this split
      const int s = hv % NV, key = t0 * kBlockN + hv * 64 + lane * bv;
      const bool mine = lane * bv < 64 && key < sq.len;
      const int page = mine ? __ldg(table + (key >> lg)) : 0;
      const bool free = hv < NV || mbar_wait(&bars[kMbVEmpty + s], (hv / NV - 1) & 1, abort_flag, 112);
      if (!__all_sync(0xffffffffu, free)) return false;
      const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_expect_tx(&bars[kMbVFull + s], boxes * bv * D * 2);
      __syncwarp();
      if (mine) {
        uint8_t* dv = smem + L::oV + s * L::kVHalf + lane * bv * 128;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(dv + c * L::kVChunk, &tmV, &bars[kMbVFull + s], c * 64, key & mask, hk, page);
      }
      __syncwarp();
      return true;
    };
    bool ok = load_k(0);
    if (ok && n_kv > 1) ok = load_k(1);
    for (int j = 0; ok && j < n_kv; ++j) {
      ok = load_v(2 * j);
      if (ok) ok = load_v(2 * j + 1);
      if (ok && j + 2 < n_kv) ok = load_k(j + 2);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc_s = make_idesc_bf16(kBlockM, kBlockN, 0, 0);
    constexpr uint32_t idesc_pv = make_idesc_bf16(kBlockM, D, 0, 1);
    constexpr uint32_t r_layout = RP == 16 ? kSwizzle32B : kSwizzle64B;
    constexpr uint32_t r_sbo = 8 * RP * 2;
    bool ok = mbar_wait(&bars[kMbQFull], 0, abort_flag, 211);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (ok && graph && n_t[i] > 0) ok = mbar_wait(&bars[kMbRqReady + i], 0, abort_flag, 212);

    // S_i(j); the last user of K(j) releases its stage
    auto issue_s = [&](int i, int j) {
      const int b = j & 1;
      const uint32_t sQ = smem_u32(smem + L::oQ + i * L::kQBytes);
      const uint32_t sK = smem_u32(smem + L::oK + b * L::kKBytes);
      const uint32_t tS = tmem + 256 + 128 * i;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = (kk >> 2) * L::kChunk + (kk & 3) * 32;
        mma_ss(tS, make_sdesc(sQ + off, 16, 1024, kSwizzle128B), make_sdesc(sK + off, 16, 1024, kSwizzle128B), idesc_s,
               kk > 0);
      }
      if (graph) {
        const uint32_t sHi = smem_u32(smem + L::oRq + i * L::kRBytes);
        const uint32_t sLo = smem_u32(smem + L::oRqLo + i * L::kRBytes);
        const uint32_t sRk = smem_u32(smem + L::oRk + b * L::kRBytes);
#pragma unroll
        for (int kk = 0; kk < RP / 16; ++kk) {
          const uint64_t rk = make_sdesc(sRk + kk * 32, 16, r_sbo, r_layout);
          mma_ss(tS, make_sdesc(sHi + kk * 32, 16, r_sbo, r_layout), rk, idesc_s, 1);
          mma_ss(tS, make_sdesc(sLo + kk * 32, 16, r_sbo, r_layout), rk, idesc_s, 1);
        }
      }
      mma_commit(&bars[kMbSFull + i]);
      if (i == 1 || j >= n_t[1]) mma_commit(&bars[kMbKEmpty + b]);
    };
    auto wait_k = [&](int j) -> bool {
      if (!mbar_wait_spin(&bars[kMbKFull + (j & 1)], (j >> 1) & 1, abort_flag, 213)) return false;
      tc_fence_after();
      return true;
    };

    if (ok) ok = wait_k(0);
    if (ok) {
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (n_t[i] > 0) issue_s(i, 0);
      }
      __syncwarp();
    }
    for (int j = 0; ok && j < n_kv; ++j) {
      const int va = 2 * j % NV, vb = (2 * j + 1) % NV;
      if (!mbar_wait_spin(&bars[kMbVFull + va], (2 * j / NV) & 1, abort_flag, 215)) break;
      if (!mbar_wait_spin(&bars[kMbVFull + vb], ((2 * j + 1) / NV) & 1, abort_flag, 215)) break;
      if (j + 1 < n_kv && !wait_k(j + 1)) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (j >= n_t[i]) continue;
        if (!mbar_wait_spin(&bars[kMbPFull + i], j & 1, abort_flag, 214)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t tO = tmem + 128 * i;
          const uint32_t tP = tmem + 256 + 128 * i;
#pragma unroll
          for (int kk = 0; kk < kBlockN / 16; ++kk) {
            const uint32_t sV = smem_u32(smem + L::oV + (kk < 4 ? va : vb) * L::kVHalf) + (kk & 3) * 2048;
            mma_ts(tO, tP + kk * 8, make_sdesc(sV, L::kVChunk, 1024, kSwizzle128B), idesc_pv,
                   (j > 0 || kk > 0) ? 1u : 0u);
          }
          if (j + 1 < n_t[i]) issue_s(i, j + 1);
        }
        __syncwarp();
      }
      if (elect_one()) {
        mma_commit(&bars[kMbVEmpty + va]);
        mma_commit(&bars[kMbVEmpty + vb]);
      }
      __syncwarp();
    }
    if (ok && elect_one()) mma_commit(&bars[kMbAllDone]);
  } else {
    // ------------------------------------------------------------ softmax (warpgroup i = query tile i)
    const int wi = warp >> 2;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + 128 * wi + lane_base;
    const uint32_t tSrow = tmem + 256 + 128 * wi + lane_base;
    const int t = tid & 127;
    const int q_local = q0 + wi * kBlockM + t;
    const int n_my = wi ? n_t[1] : n_t[0];
    const float sl2 = p.scale_log2;
    bool ok = true;

    if (graph && n_my > 0) {
      // R~_q = R_q * gs/scale as hi (in place) + lo, element-wise and so independent of the swizzle
      ok = mbar_wait(&bars[kMbQFull], 0, abort_flag, 311);
      if (ok) {
        const float f = __ldg(p.gs + h) / p.scale;
        uint4* rrow = reinterpret_cast<uint4*>(smem + L::oRq + wi * L::kRBytes + t * RP * 2);
        uint4* lrow = reinterpret_cast<uint4*>(smem + L::oRqLo + wi * L::kRBytes + t * RP * 2);
#pragma unroll
        for (int u = 0; u < RP / 8; ++u) {
          uint32_t hi[4], lo[4];
          split_bias(rrow[u], f, hi, lo);
          rrow[u] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          lrow[u] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kMbRqReady + wi]);
    }

    // keys of this split that the row sees, counted from its first
    const int limit = (p.causal ? min(sq.len, past + q_local + 1) : sq.len) - t0 * kBlockN;
    const int live = sq.len - t0 * kBlockN;  // keys that exist
    float m_use = -INFINITY, m_true = -INFINITY, l = 0.f;
    uint32_t r[128];
    for (int j = 0; ok && j < n_my; ++j) {
      if (!mbar_wait(&bars[kMbSFull + wi], j & 1, abort_flag, 312)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tSrow + 32 * c, r + 32 * c);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_wait32(r + 32 * c);

      const int nvalid = limit - j * kBlockN;
      float m8[8];  // independent chains
#pragma unroll
      for (int k = 0; k < 8; ++k) m8[k] = -INFINITY;
      if (nvalid >= kBlockN) {
#pragma unroll
        for (int k = 0; k < 128; ++k) m8[k & 7] = fmaxf(m8[k & 7], __uint_as_float(r[k]));
      } else {
#pragma unroll
        for (int k = 0; k < 128; ++k) {
          const float x = k < nvalid ? __uint_as_float(r[k]) : -INFINITY;
          r[k] = __float_as_uint(x);
          m8[k & 7] = fmaxf(m8[k & 7], x);
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
      mx *= sl2;
      m_true = fmaxf(m_true, mx);
      float alpha = 1.f;
      bool rescale = false;
      if (m_true - m_use > 8.f || m_use == -INFINITY) {
        alpha = (m_use == -INFINITY) ? 0.f : ex2(m_use - m_true);
        rescale = (j > 0);
        m_use = m_true;
      }
      const float mb = (m_use == -INFINITY) ? 0.f : m_use;
      float rs4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 128; k += 2) {
        const float p0 = ex2(fmaf(__uint_as_float(r[k]), sl2, -mb));
        const float p1 = ex2(fmaf(__uint_as_float(r[k + 1]), sl2, -mb));
        rs4[(k >> 1) & 3] += p0 + p1;
        r[k >> 1] = pack_bf16(p0, p1);
      }
      l = l * alpha + ((rs4[0] + rs4[1]) + (rs4[2] + rs4[3]));
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_st16(tSrow + 16 * c, r + 16 * c);
      // O_i += P_i(j-1) V(j-1) is complete (covered by the S_i(j) commit): rescale O_i if needed
      if (j > 0 && __any_sync(0xffffffffu, rescale)) {
        const float a = rescale ? alpha : 1.f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * c, o);
          tmem_ld_wait32(o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * a);
          tmem_st32(tO + 32 * c, o);
        }
      }
      const int nlive = live - j * kBlockN;
      if (nlive < kBlockN) {
        // the sequence's last tile: V rows that no key owns become zero (both warpgroups write the same
        // zeros; nothing refills these stages, so their barriers keep the phase that is waited for)
#pragma unroll 1
        for (int hv = 2 * j; hv < 2 * j + 2; ++hv) {
          if (!mbar_wait(&bars[kMbVFull + hv % NV], (hv / NV) & 1, abort_flag, 313)) ok = false;
          const int first = max(0, nlive - (hv & 1) * 64);
          uint8_t* sv = smem + L::oV + (hv % NV) * L::kVHalf;
          for (int e = t; ok && e < (64 - first) * 8 * (D / 64); e += 128) {
            const int c = e / ((64 - first) * 8), x = e % ((64 - first) * 8);
            *reinterpret_cast<uint4*>(sv + c * L::kVChunk + first * 128 + x * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kMbPFull + wi]);
    }

    const bool row_ok = q_local < sq.n;
    if (ok && n_my > 0 && mbar_wait(&bars[kMbAllDone], 0, abort_flag, 314)) {
      tc_fence_after();
      const float corr = (m_use == -INFINITY) ? 0.f : ex2(m_use - m_true);
      const float l_true = l * corr;
      const int row0 = q0 + wi * kBlockM + (warp & 3) * 32;
      if (it.ns == 1) {
        const float inv = corr / (l_true + kEps);
        __nv_bfloat16* o0 = p.out + static_cast<int64_t>(sq.q0 + row0) * p.o_st + h * p.o_sh;
        store_o_rows<D>(smem + L::oK + warp * 32 * 64, tO, inv, o0, p.o_st, sq.n - row0);
        if (row_ok && p.lse) p.lse[h * p.lse_sh + sq.q0 + q_local] = (m_true + lg2(l_true + kEps)) * kLn2;
      } else {
        const int64_t w = (static_cast<int64_t>(sq.q0 + q_local) * p.H + h) * p.ns + it.split;
        if (row_ok) p.ws_ml[w] = make_float2(m_true, l_true);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * c, o);
          tmem_ld_wait32(o);
          if (row_ok) {
            float4* dst = reinterpret_cast<float4*>(p.ws_acc + w * D + 32 * c);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              dst[k] = make_float4(__uint_as_float(o[4 * k]) * corr, __uint_as_float(o[4 * k + 1]) * corr,
                                   __uint_as_float(o[4 * k + 2]) * corr, __uint_as_float(o[4 * k + 3]) * corr);
          }
        }
      }
    } else if (n_my == 0 && row_ok) {
      write_none(q_local);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct ManyMaps {
  CUtensorMap q, k, v, rq, rk;
};

template <int D, int RP>
cudaError_t launch_paged_many_t(const ManyMaps& m, const PagedAttnParams& p, cudaStream_t stream) {
  using L = ManySmem<D, RP>;
  auto kern = fna2_paged_many_kernel<D, RP>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(p.H * p.many_items), kFwdThreads, L::kTotal, stream, m.q, m.k, m.v, m.rq, m.rk, p);
}

inline cudaError_t launch_paged_many(const ManyMaps& m, const PagedAttnParams& p, int D, cudaStream_t stream) {
  if (D == 64) return p.RP == 16 ? launch_paged_many_t<64, 16>(m, p, stream) : launch_paged_many_t<64, 32>(m, p, stream);
  return p.RP == 16 ? launch_paged_many_t<128, 16>(m, p, stream) : launch_paged_many_t<128, 32>(m, p, stream);
}

}  // namespace fna2
