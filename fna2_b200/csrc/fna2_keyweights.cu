// Attention weight that each cached key received:
//   w[b, kh, j] += sum over query heads h of KV head kh and new tokens i that
//                  see key j of exp(S[h,i,j] - LSE[h,i])
// with S and LSE as in the paged attention (fna2_paged.cu).
//
// Key-stationary on the tensor cores: the transposed scores S^T = [K | R_k | R_k]
// [Q | R~_q hi | R~_q lo]^T put a key on every TMEM lane, so the thread that owns
// a key sums its weights over the columns in a register: no reduction between
// threads, no atomics on the result, which does not depend on timing.  An item is a
// pair of 128-key tiles of one (sequence, KV head); its units are the (query head,
// tile of QT queries) that see it.  One persistent CTA per SM draws items from a
// counter and streams their units through a two-stage ring: Q, R~_q hi and lo, and
// the R_k rows of that head for its keys.  QT is 64 when no sequence has more
// queries (K is then double-buffered: an item is only as many units as there are
// heads), else 128.
//   warps 0-3 / 4-7  sum key tile 0 / 1 (thread t = key t = TMEM lane t)
//   warp 8           draws items, TMA producer (K and R_k page by page, as in
//                    fna2_paged_many.cu)
//   warp 9           TMEM allocation, MMA issue; each key tile has 256 / QT TMEM
//                    buffers, so its next MMAs run while a unit is summed
// The LSE has a ring of its own: with it in the operands' stages, a unit's loads
// waited for the sums two units before (4200 clk per unit at QT = 128).
// A small kernel first writes R~_q hi / lo rows and the log2-domain LSE.
// Bound: one exp2 per (key, query, head), 16 per clock and SM: 2 x 128 x 128 of them
// take 2048 clk per unit, the 2 x (D + 2 r_pad)/16 MMAs about 1300.
#include "fna2_paged.cuh"

namespace fna2 {

struct KeyWeightsParams {
  PagedPool kv;
  PagedBounds bd;
  int H, G, RP, causal;
  float scale, scale_log2;
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const __nv_bfloat16* rq;
  int64_t rq_st, rq_sh;
  const float* gs;
  const float* lse;  // [H][lse_sh]
  int64_t lse_sh;
  float* kw;
  int64_t kw_sb, kw_sh;
  __nv_bfloat16* rq2;  // workspace: [T][H_G][2 RP] R~_q hi, lo
  float* lse2;         // workspace: [H][T] -LSE * log2(e), -inf for a row without weight
  int* next;           // workspace: item counter, zeroed by the prep kernel
};

// R~_q = gs/scale * R_q as hi + lo, columns [rank, RP) zero; -LSE in the log2 domain.
__global__ void __launch_bounds__(256) fna2_key_weights_prep_kernel(const KeyWeightsParams p) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e == 0) *p.next = 0;
  const int r8 = p.RP / 8;
  const int64_t n_r = static_cast<int64_t>(p.bd.T) * p.kv.hg * r8, n_l = static_cast<int64_t>(p.bd.T) * p.H;
  if (e < n_r) {
    const int c = static_cast<int>(e % r8) * 8, h = static_cast<int>(e / r8 % p.kv.hg);
    const int64_t t = e / r8 / p.kv.hg;
    uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
    if (c < p.kv.rank)
      split_bias(*reinterpret_cast<const uint4*>(p.rq + t * p.rq_st + h * p.rq_sh + c), __ldg(p.gs + h) / p.scale, hi, lo);
    __nv_bfloat16* dst = p.rq2 + (t * p.kv.hg + h) * 2 * p.RP + c;
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(dst + p.RP) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  if (e < n_l) {
    const int64_t h = e / p.bd.T, t = e % p.bd.T;
    const float v = p.lse[h * p.lse_sh + t];
    p.lse2[e] = v == -INFINITY ? v : -v * kLog2e;
  }
}

constexpr int kKwThreads = 320;

template <int D, int RP, int QT>
struct KwSmem {
  static constexpr int kTile = 128 * D * 2;    // K tile
  static constexpr int kRTile = 128 * RP * 2;  // R_k of a key tile
  static constexpr int kQTile = QT * D * 2;
  static constexpr int kRqTile = QT * RP * 2;  // R~_q hi or lo
  static constexpr int kChunk = 128 * 128;     // 64 columns of a 128-row tile
  static constexpr int kQChunk = QT * 128;
  static constexpr int kKStages = QT == 64 ? 2 : 1;
  static constexpr int oK = 0;                                // kKStages x key tiles 0, 1
  static constexpr int oStage = oK + kKStages * 2 * kTile;    // 2 x [Q | R_k 0, 1 | R~_q hi, lo]
  static constexpr int sQ = 0, sRk = kQTile, sRq = sRk + 2 * kRTile;
  static constexpr int kStage = sRq + 2 * kRqTile;
  static constexpr int kBufs = 256 / QT;                      // TMEM buffers per key tile
  static constexpr int oLse = oStage + 2 * kStage;            // 4 x -LSE of a unit
  static constexpr int oBar = oLse + 4 * QT * 4;
  static constexpr int oMisc = oBar + 32 * 8;
  static constexpr int oItem = oMisc + 16;                    // kKStages x KwItem
  static constexpr int kUsed = oItem + kKStages * 32;
  static constexpr int kTotal = kUsed + 1024;
  static_assert(kTotal <= kMaxDynamicSmem, "shared memory budget");
  static_assert(kStage % 1024 == 0, "swizzle atoms stay aligned");
};

enum KwBar {
  kWbKFull = 0,    // +K stage: K and the item's description
  kWbKEmpty = 2,   // +K stage: its MMAs are done, every sum warp has left the item (1 + 8 arrivals)
  kWbFull = 4,     // +stage: the unit's operands
  kWbEmpty = 6,    // +stage: MMAs that read it are done
  kWbLFull = 8,    // +LSE slot
  kWbLEmpty = 12,  // +LSE slot (8 arrivals)
  kWbSFull = 16,   // +4 tile + buffer
  kWbSEmpty = 24,  // +4 tile + buffer (one arrival per warp)
};

struct KwItem {
  int b, kh, k0, len, n, u0, per_head, n_units;  // n_units < 0: no more items; u0: first query tile
};

// Item `idx`: (pair of key tiles, KV head) of the sequences in packing order, KV heads of a pair
// together, early keys (which the most queries see) first.  Called by a whole warp.
__device__ __forceinline__ KwItem kw_item(const KeyWeightsParams& p, int idx, int lane, int QT) {
  KwItem it;
  it.n_units = -1;
  int carry = 0;
  for (int base = 0; base < p.bd.B; base += 32) {
    const int b = base + lane;
    PagedSeq s{0, 0, 0, false};
    int cnt = 0;
    if (b < p.bd.B) {
      s = paged_seq(p.bd, b);
      if (!s.ok) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
      if (s.n > 0) cnt = (s.len + 2 * kBlockN - 1) / (2 * kBlockN) * p.kv.hkv;
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
      it.b = base + src;
      it.kh = local % p.kv.hkv;
      it.k0 = local / p.kv.hkv * 2 * kBlockN;
      it.len = __shfl_sync(0xffffffffu, s.len, src);
      it.n = __shfl_sync(0xffffffffu, s.n, src);
      const int n_qt = (it.n + QT - 1) / QT;
      it.u0 = p.causal ? min(n_qt, max(0, it.k0 - (it.len - it.n)) / QT) : 0;  // earlier tokens see none of these keys
      it.per_head = n_qt - it.u0;
      it.n_units = it.per_head * p.G;
      return it;
    }
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  return it;
}

// Sum over the QT columns of this thread's lane of 2^(sl2 S - LSE); MASK: of columns [lo, hi) only.
// (Two copies: masks cost 5 instructions per column.)
template <int QT, bool MASK>
__device__ __forceinline__ float kw_sum(uint32_t t_addr, const float4* lse4, float2 sl2, int lo, int hi) {
  float2 a[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t r[2][32];
  tmem_ld32(t_addr, r[0]);
#pragma unroll
  for (int c = 0; c < QT / 32; ++c) {
    uint32_t* x = r[c & 1];
    tmem_ld_wait32(x);
    if (c + 1 < QT / 32) tmem_ld32(t_addr + 32 * (c + 1), r[(c + 1) & 1]);
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      const float4 l = lse4[8 * c + k / 4];
      const float2 y0 = __ffma2_rn(f32x2(x[k], x[k + 1]), sl2, make_float2(l.x, l.y));
      const float2 y1 = __ffma2_rn(f32x2(x[k + 2], x[k + 3]), sl2, make_float2(l.z, l.w));
      float2 e0 = make_float2(ex2(y0.x), ex2(y0.y)), e1 = make_float2(ex2(y1.x), ex2(y1.y));
      if (MASK) {
        const int col = 32 * c + k;
        e0.x = col >= lo && col < hi ? e0.x : 0.f;
        e0.y = col + 1 >= lo && col + 1 < hi ? e0.y : 0.f;
        e1.x = col + 2 >= lo && col + 2 < hi ? e1.x : 0.f;
        e1.y = col + 3 >= lo && col + 3 < hi ? e1.y : 0.f;
      }
      a[0] = __fadd2_rn(a[0], e0);
      a[1] = __fadd2_rn(a[1], e1);
    }
  }
  return (a[0].x + a[0].y) + (a[1].x + a[1].y);
}

template <int D, int RP, int QT>
__global__ void __launch_bounds__(kKwThreads, 1)
    fna2_key_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmRq, const __grid_constant__ CUtensorMap tmRk,
                            const KeyWeightsParams p) {
  using L = KwSmem<D, RP, QT>;
  constexpr int KS = L::kKStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::oMisc + 4);
  volatile KwItem* items = reinterpret_cast<volatile KwItem*>(smem + L::oItem);
  const int warp = warp_id(), lane = lane_id(), tid = threadIdx.x;

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kWbKFull + s], 1);
      mbar_init(&bars[kWbKEmpty + s], 9);
      mbar_init(&bars[kWbFull + s], 1);
      mbar_init(&bars[kWbEmpty + s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars[kWbLFull + s], 1);
      mbar_init(&bars[kWbLEmpty + s], 8);
    }
    for (int s = 0; s < 8; ++s) {
      mbar_init(&bars[kWbSFull + s], 1);
      mbar_init(&bars[kWbSEmpty + s], 4);
    }
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
    }
    const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
    const int bk = min(1 << lg, kBlockN);  // rows of a box; lane l owns box l of the two key tiles (at most 16)
    const int tile = lane * bk / kBlockN, row = lane * bk % kBlockN;
    int gu = 0;  // units so far
    for (int n = 0;; ++n) {
      const int ks = n % KS;
      int idx = 0;
      if (lane == 0) idx = atomicAdd(p.next, 1);
      idx = __shfl_sync(0xffffffffu, idx, 0);
      const KwItem it = kw_item(p, idx, lane, QT);
      const bool free = n < KS || mbar_wait(&bars[kWbKEmpty + ks], (n / KS - 1) & 1, abort_flag, 120);
      if (!__all_sync(0xffffffffu, free)) break;
      const int key = it.k0 + lane * bk;
      const bool mine = it.n_units >= 0 && lane * bk < 2 * kBlockN && key < it.len;
      const int page = mine ? __ldg(p.kv.table + it.b * p.kv.table_sb + (key >> lg)) : 0;
      const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) {  // (the arrival also publishes the description)
        volatile KwItem* d = items + ks;
        d->b = it.b, d->kh = it.kh, d->k0 = it.k0, d->len = it.len, d->n = it.n, d->u0 = it.u0;
        d->per_head = it.per_head, d->n_units = it.n_units;
        mbar_expect_tx(&bars[kWbKFull + ks], boxes * bk * D * 2);
      }
      __syncwarp();
      if (it.n_units < 0) break;
      if (mine) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + L::oK + (2 * ks + tile) * L::kTile + c * L::kChunk + row * 128, &tmK,
                      &bars[kWbKFull + ks], c * 64, key & mask, it.kh, page);
      }
      __syncwarp();
      const int q0 = __ldg(p.bd.cu + it.b);
      bool ok = true;
      for (int u = 0; u < it.n_units; ++u, ++gu) {
        const int s = gu & 1, h = it.kh * p.G + u / it.per_head;
        const int i0 = (it.u0 + u % it.per_head) * QT, tok = q0 + i0;
        const bool graph = h < p.kv.hg;
        uint8_t* st = smem + L::oStage + s * L::kStage;
        // this unit's -LSE (columns past the end: -inf, which adds 0)
        float lse[QT / 32];
#pragma unroll
        for (int k = 0; k < QT / 32; ++k) {
          const int i = lane + 32 * k;
          lse[k] = i0 + i < it.n ? p.lse2[static_cast<int64_t>(h) * p.bd.T + tok + i] : -INFINITY;
        }
        const bool room = (gu < 4 || mbar_wait(&bars[kWbLEmpty + (gu & 3)], ((gu >> 2) - 1) & 1, abort_flag, 122)) &&
                          (gu < 2 || mbar_wait(&bars[kWbEmpty + s], ((gu >> 1) - 1) & 1, abort_flag, 121));
        ok = __all_sync(0xffffffffu, room);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < QT / 32; ++k)
          reinterpret_cast<float*>(smem + L::oLse)[(gu & 3) * QT + lane + 32 * k] = lse[k];
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars[kWbLFull + (gu & 3)]);
          mbar_expect_tx(&bars[kWbFull + s], QT * (D + (graph ? 2 * RP : 0)) * 2 + (graph ? boxes * bk * RP * 2 : 0));
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(st + L::sQ + c * L::kQChunk, &tmQ, &bars[kWbFull + s], c * 64, tok, h, 0);
          if (graph) {
            tma_load_4d(st + L::sRq, &tmRq, &bars[kWbFull + s], 0, tok, h, 0);
            tma_load_4d(st + L::sRq + L::kRqTile, &tmRq, &bars[kWbFull + s], RP, tok, h, 0);
          }
        }
        __syncwarp();
        if (mine && graph)
          tma_load_4d(st + L::sRk + tile * L::kRTile + row * RP * 2, &tmRk, &bars[kWbFull + s], 0, key & mask, h, page);
        __syncwarp();
      }
      if (!ok) break;
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = make_idesc_bf16(kBlockN, QT, 0, 0);
    constexpr uint32_t r_layout = RP == 16 ? kSwizzle32B : kSwizzle64B;
    constexpr uint32_t r_sbo = 8 * RP * 2;
    constexpr int NB = L::kBufs;
    int gu = 0, used[2] = {0, 0};
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const int ks = n % KS;
      if (!mbar_wait(&bars[kWbKFull + ks], (n / KS) & 1, abort_flag, 221)) break;
      const int n_units = items[ks].n_units, per_head = items[ks].per_head, h0 = items[ks].kh * p.G;
      const int tiles = items[ks].k0 + kBlockN < items[ks].len ? 2 : 1;
      if (n_units < 0) break;
      for (int u = 0; ok && u < n_units; ++u, ++gu) {
        const int s = gu & 1;
        const bool graph = h0 + u / per_head < p.kv.hg;
        if (!mbar_wait_spin(&bars[kWbFull + s], (gu >> 1) & 1, abort_flag, 222)) {
          ok = false;
          break;
        }
        const uint32_t st = smem_u32(smem + L::oStage + s * L::kStage);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= tiles) continue;
          const int buf = used[i] % NB;
          if (used[i] >= NB && !mbar_wait_spin(&bars[kWbSEmpty + 4 * i + buf], (used[i] / NB - 1) & 1, abort_flag, 223)) {
            ok = false;
            break;
          }
          ++used[i];
          tc_fence_after();
          if (elect_one()) {
            const uint32_t tS = tmem + 256 * i + QT * buf;
            const uint32_t sK = smem_u32(smem + L::oK + (2 * ks + i) * L::kTile);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_ss(tS, make_sdesc(sK + (kk >> 2) * L::kChunk + (kk & 3) * 32, 16, 1024, kSwizzle128B),
                     make_sdesc(st + L::sQ + (kk >> 2) * L::kQChunk + (kk & 3) * 32, 16, 1024, kSwizzle128B), idesc,
                     kk > 0);
            if (graph) {
#pragma unroll
              for (int kk = 0; kk < RP / 16; ++kk) {
                const uint64_t rk = make_sdesc(st + L::sRk + i * L::kRTile + kk * 32, 16, r_sbo, r_layout);
                mma_ss(tS, rk, make_sdesc(st + L::sRq + kk * 32, 16, r_sbo, r_layout), idesc, 1);
                mma_ss(tS, rk, make_sdesc(st + L::sRq + L::kRqTile + kk * 32, 16, r_sbo, r_layout), idesc, 1);
              }
            }
            mma_commit(&bars[kWbSFull + 4 * i + buf]);
            if (i == tiles - 1) mma_commit(&bars[kWbEmpty + s]);
          }
          __syncwarp();
        }
      }
      if (ok && elect_one()) mma_commit(&bars[kWbKEmpty + ks]);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ sums (warpgroup i = key tile i)
    const int wi = warp >> 2;
    const uint32_t t_lane = tmem + 256 * wi + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    int gu = 0, used = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const int ks = n % KS;
      if (!mbar_wait(&bars[kWbKFull + ks], (n / KS) & 1, abort_flag, 320)) break;
      const int n_units = items[ks].n_units, per_head = items[ks].per_head, u0 = items[ks].u0, nq = items[ks].n;
      const int len = items[ks].len, tile0 = items[ks].k0 + wi * kBlockN, j = tile0 + (tid & 127), past = len - nq;
      if (n_units < 0) break;
      const bool mine = tile0 < len;
      float* dst = p.kw + items[ks].b * p.kw_sb + items[ks].kh * p.kw_sh + j;
      float w = mine && j < len ? *dst : 0.f;
      for (int u = 0; u < n_units; ++u, ++gu) {
        const int ls = gu & 3, buf = used % L::kBufs;
        if (!mbar_wait(&bars[kWbLFull + ls], (gu >> 2) & 1, abort_flag, 321) ||
            (mine && !mbar_wait(&bars[kWbSFull + 4 * wi + buf], (used / L::kBufs) & 1, abort_flag, 322))) {
          ok = false;
          break;
        }
        if (mine) {
          ++used;
          tc_fence_after();
          const int i0 = (u0 + u % per_head) * QT;
          const float4* lse4 = reinterpret_cast<const float4*>(smem + L::oLse + ls * QT * 4);
          // columns [first, nq - i0) belong to queries that see the key; a NaN score of another sequence's
          // query is never read into a sum
          const int first = p.causal ? j - past - i0 : 0;
          const bool whole = (!p.causal || tile0 + kBlockN - 1 <= past + i0) && i0 + QT <= nq;
          w += whole ? kw_sum<QT, false>(t_lane + QT * buf, lse4, sl2, 0, 0)
                     : kw_sum<QT, true>(t_lane + QT * buf, lse4, sl2, first, nq - i0);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          if (mine) mbar_arrive(&bars[kWbSEmpty + 4 * wi + buf]);
          mbar_arrive(&bars[kWbLEmpty + ls]);
        }
      }
      if (ok && mine && j < len) *dst = w;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kWbKEmpty + ks]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct KwMaps {
  CUtensorMap q, k, rq, rk;
};

// Queries per unit.
inline int kw_query_tile(const KeyWeightsParams& p) { return p.bd.max_q <= 64 ? 64 : 128; }

template <int D, int RP, int QT>
cudaError_t launch_key_weights_t(const KwMaps& m, const KeyWeightsParams& p, cudaStream_t stream) {
  using L = KwSmem<D, RP, QT>;
  auto kern = fna2_key_weights_kernel<D, RP, QT>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed);
  if (e != cudaSuccess) return e;
  const int64_t n = static_cast<int64_t>(p.bd.T) * std::max<int64_t>(p.H, static_cast<int64_t>(p.kv.hg) * p.RP / 8);
  fna2_key_weights_prep_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t items = static_cast<int64_t>(p.bd.B) * p.kv.hkv * ((p.bd.max_k + 2 * kBlockN - 1) / (2 * kBlockN));
  kern<<<static_cast<unsigned>(std::min<int64_t>(items, kSms)), kKwThreads, L::kTotal, stream>>>(m.q, m.k, m.rq, m.rk, p);
  return cudaGetLastError();
}

template <int D, int RP>
cudaError_t launch_key_weights_r(const KwMaps& m, const KeyWeightsParams& p, cudaStream_t stream) {
  return kw_query_tile(p) == 64 ? launch_key_weights_t<D, RP, 64>(m, p, stream)
                                : launch_key_weights_t<D, RP, 128>(m, p, stream);
}

inline cudaError_t launch_key_weights(const KwMaps& m, const KeyWeightsParams& p, int D, cudaStream_t stream) {
  if (D == 64) return p.RP == 16 ? launch_key_weights_r<64, 16>(m, p, stream) : launch_key_weights_r<64, 32>(m, p, stream);
  return p.RP == 16 ? launch_key_weights_r<128, 16>(m, p, stream) : launch_key_weights_r<128, 32>(m, p, stream);
}

}  // namespace fna2
