// Attention weight that each cached key received:
//   w[b, kh, j] += sum over query heads h of KV head kh and new tokens i that
//                  see key j of exp(S[h,i,j] - LSE[h,i])
// with S and LSE as in the paged attention (fna2_paged.cu).
//
// Key-stationary on the tensor cores: the transposed scores S^T = [K | R_k | R_k]
// [Q | R~_q hi | R~_q lo]^T put a key on every TMEM lane, so the thread that owns
// a key sums its weights over the columns in a register: no reduction between
// threads, no atomics, a result that does not depend on timing.  A CTA owns a
// pair of 128-key tiles of one (sequence, KV head) and streams (query head, tile of
// QT queries) units through a two-stage ring: Q, R~_q hi and lo, and the R_k rows
// of that head for its keys.  QT is 64 when no sequence has more queries, else 128.
//   warps 0-3 / 4-7  sum key tile 0 / 1 (thread t = key t = TMEM lane t)
//   warp 8           TMA producer (K and R_k page by page, as in fna2_paged_many.cu)
//   warp 9           TMEM allocation, MMA issue; S^T of key tile i, unit u in the
//                    TMEM buffer 2 i + (u & 1), so a tile's MMAs run while the
//                    previous unit is summed
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
  float* lse2;         // workspace: [H][T] LSE * log2(e), +inf for a row without weight
  int qt;              // queries per unit
};

// R~_q = gs/scale * R_q as hi + lo, columns [rank, RP) zero; LSE in the log2 domain.
__global__ void __launch_bounds__(256) fna2_key_weights_prep_kernel(const KeyWeightsParams p) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
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
    p.lse2[e] = v == -INFINITY ? INFINITY : v * kLog2e;
  }
}

constexpr int kKwThreads = 320;

template <int D, int RP>
struct KwSmem {
  static constexpr int kTile = 128 * D * 2;   // K tile, Q tile
  static constexpr int kRTile = 128 * RP * 2;  // R_k of a key tile; R~_q hi or lo
  static constexpr int kChunk = 128 * 128;     // 64 columns of a 128-row tile
  static constexpr int oK = 0;                               // key tiles 0, 1
  static constexpr int oStage = oK + 2 * kTile;              // 2 x [Q | R_k 0, 1 | R~_q hi, lo | LSE]
  static constexpr int sQ = 0, sRk = kTile, sRq = sRk + 2 * kRTile, sLse = sRq + 2 * kRTile;
  static constexpr int kStage = sLse + 1024;
  static constexpr int oBar = oStage + 2 * kStage;
  static constexpr int oMisc = oBar + 16 * 8;
  static constexpr int kUsed = oMisc + 16;
  static constexpr int kTotal = kUsed + 1024;
  static_assert(kTotal <= kMaxDynamicSmem, "shared memory budget");
};

enum KwBar {
  kWbKFull = 0,
  kWbFull = 1,    // +stage: the unit's operands
  kWbEmpty = 3,   // +stage: MMAs that read it are done, and its LSE has been read (1 + 8 arrivals)
  kWbSFull = 5,   // +2 tile + buffer
  kWbSEmpty = 9,  // +2 tile + buffer (one arrival per warp)
};

template <int D, int RP>
__global__ void __launch_bounds__(kKwThreads, 1)
    fna2_key_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmRq, const __grid_constant__ CUtensorMap tmRk,
                            const KeyWeightsParams p) {
  using L = KwSmem<D, RP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::oMisc + 4);
  const int warp = warp_id(), lane = lane_id(), tid = threadIdx.x;
  const int kh = blockIdx.x, b = blockIdx.z, k0 = blockIdx.y * 2 * kBlockN;
  const PagedSeq sq = paged_seq(p.bd, b);
  if (!sq.ok && tid == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
  if (k0 >= sq.len || sq.n == 0) return;
  const int past = sq.len - sq.n, QT = p.qt;
  const bool two = k0 + kBlockN < sq.len;  // the second key tile has keys
  // query tiles [u0, n_qt): earlier tokens see none of these keys
  const int n_qt = (sq.n + QT - 1) / QT, u0 = p.causal ? min(n_qt, max(0, k0 - past) / QT) : 0;
  const int per_head = n_qt - u0, n_units = per_head * p.G;
  if (n_units == 0) return;

  if (tid == 0) {
    mbar_init(&bars[kWbKFull], 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kWbFull + s], 1);
      mbar_init(&bars[kWbEmpty + s], two ? 9 : 5);
    }
    for (int s = 0; s < 4; ++s) {
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
  const int hg_local = p.kv.hg - kh * p.G;  // heads of the group below this carry the bias

  if (warp == 8) {
    // ------------------------------------------------------------ producer
    const int* table = p.kv.table + b * p.kv.table_sb;
    const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
    const int bk = min(1 << lg, kBlockN);  // rows of a box; lane l owns box l of the two key tiles (at most 16)
    const int key = k0 + lane * bk;
    const bool mine = lane * bk < 2 * kBlockN && key < sq.len;
    const int page = mine ? __ldg(table + (key >> lg)) : 0;
    const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
    const int tile = lane * bk / kBlockN, row = lane * bk % kBlockN;
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      mbar_expect_tx(&bars[kWbKFull], boxes * bk * D * 2);
    }
    __syncwarp();
    if (mine) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_load_4d(smem + L::oK + tile * L::kTile + c * L::kChunk + row * 128, &tmK, &bars[kWbKFull], c * 64,
                    key & mask, kh, page);
    }
    for (int u = 0; u < n_units; ++u) {
      const int s = u & 1, g = u / per_head, h = kh * p.G + g;
      const int i0 = (u0 + u % per_head) * QT, tok = sq.q0 + i0;
      const bool graph = g < hg_local;
      uint8_t* st = smem + L::oStage + s * L::kStage;
      // this unit's LSE (columns past the end: +inf, which adds 0)
      float lse[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = lane + 32 * k;
        lse[k] = i < QT && i0 + i < sq.n ? p.lse2[static_cast<int64_t>(h) * p.bd.T + tok + i] : INFINITY;
      }
      const bool free = u < 2 || mbar_wait(&bars[kWbEmpty + s], ((u >> 1) - 1) & 1, abort_flag, 121);
      if (!__all_sync(0xffffffffu, free)) break;
#pragma unroll
      for (int k = 0; k < 4; ++k) reinterpret_cast<float*>(st + L::sLse)[lane + 32 * k] = lse[k];
      __syncwarp();
      if (lane == 0) {  // (the arrival also publishes the LSE)
        mbar_expect_tx(&bars[kWbFull + s], QT * (D + (graph ? 2 * RP : 0)) * 2 + (graph ? boxes * bk * RP * 2 : 0));
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(st + L::sQ + c * L::kChunk, &tmQ, &bars[kWbFull + s], c * 64, tok, h, 0);
        if (graph) {
          tma_load_4d(st + L::sRq, &tmRq, &bars[kWbFull + s], 0, tok, h, 0);
          tma_load_4d(st + L::sRq + L::kRTile, &tmRq, &bars[kWbFull + s], RP, tok, h, 0);
        }
      }
      __syncwarp();
      if (mine && graph)
        tma_load_4d(st + L::sRk + tile * L::kRTile + row * RP * 2, &tmRk, &bars[kWbFull + s], 0, key & mask, h, page);
      __syncwarp();
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc = QT == 64 ? make_idesc_bf16(kBlockN, 64, 0, 0) : make_idesc_bf16(kBlockN, 128, 0, 0);
    constexpr uint32_t r_layout = RP == 16 ? kSwizzle32B : kSwizzle64B;
    constexpr uint32_t r_sbo = 8 * RP * 2;
    bool ok = mbar_wait(&bars[kWbKFull], 0, abort_flag, 221);
    for (int u = 0; ok && u < n_units; ++u) {
      const int s = u & 1;
      const bool graph = u / per_head < hg_local;
      if (!mbar_wait_spin(&bars[kWbFull + s], (u >> 1) & 1, abort_flag, 222)) break;
      const uint32_t st = smem_u32(smem + L::oStage + s * L::kStage);
      for (int i = 0; i < (two ? 2 : 1); ++i) {
        const int buf = 2 * i + s;
        if (u >= 2 && !mbar_wait_spin(&bars[kWbSEmpty + buf], ((u >> 1) - 1) & 1, abort_flag, 223)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t tS = tmem + 128 * buf;
          const uint32_t sK = smem_u32(smem + L::oK + i * L::kTile);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * L::kChunk + (kk & 3) * 32;
            mma_ss(tS, make_sdesc(sK + off, 16, 1024, kSwizzle128B),
                   make_sdesc(st + L::sQ + off, 16, 1024, kSwizzle128B), idesc, kk > 0);
          }
          if (graph) {
#pragma unroll
            for (int kk = 0; kk < RP / 16; ++kk) {
              const uint64_t rk = make_sdesc(st + L::sRk + i * L::kRTile + kk * 32, 16, r_sbo, r_layout);
              mma_ss(tS, rk, make_sdesc(st + L::sRq + kk * 32, 16, r_sbo, r_layout), idesc, 1);
              mma_ss(tS, rk, make_sdesc(st + L::sRq + L::kRTile + kk * 32, 16, r_sbo, r_layout), idesc, 1);
            }
          }
          mma_commit(&bars[kWbSFull + buf]);
          if (i == (two ? 1 : 0)) mma_commit(&bars[kWbEmpty + s]);
        }
        __syncwarp();
      }
    }
  } else if (two || warp < 4) {
    // ------------------------------------------------------------ sums (warpgroup i = key tile i)
    const int wi = warp >> 2, j = k0 + wi * kBlockN + (tid & 127);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float sl2 = p.scale_log2;
    const int tile_last = k0 + wi * kBlockN + kBlockN - 1;
    float w = 0.f;
    bool ok = true;
    for (int u = 0; u < n_units; ++u) {
      const int s = u & 1, buf = 2 * wi + s;
      const int i0 = (u0 + u % per_head) * QT;
      if (!mbar_wait(&bars[kWbFull + s], (u >> 1) & 1, abort_flag, 321) ||
          !mbar_wait(&bars[kWbSFull + buf], (u >> 1) & 1, abort_flag, 322)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const float4* lse4 = reinterpret_cast<const float4*>(smem + L::oStage + s * L::kStage + L::sLse);
      // columns of queries that see the key start here (0: all); a NaN score of another sequence's
      // query or of a page's unused slot is never read into a sum
      const int first = p.causal ? j - past - i0 : 0;
      const bool whole = (!p.causal || tile_last <= past + i0) && i0 + QT <= sq.n;
      float a4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int c = 0; c < QT / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(tmem + 128 * buf + 32 * c + lane_base, r);
        tmem_ld_wait32(r);
        if (whole) {
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float4 l = lse4[8 * c + k / 4];
            a4[0] += ex2(fmaf(__uint_as_float(r[k]), sl2, -l.x));
            a4[1] += ex2(fmaf(__uint_as_float(r[k + 1]), sl2, -l.y));
            a4[2] += ex2(fmaf(__uint_as_float(r[k + 2]), sl2, -l.z));
            a4[3] += ex2(fmaf(__uint_as_float(r[k + 3]), sl2, -l.w));
          }
        } else {
          const int lo = first - 32 * c, hi = sq.n - i0 - 32 * c;
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float4 l = lse4[8 * c + k / 4];
            const float ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const float x = ex2(fmaf(__uint_as_float(r[k + m]), sl2, -ll[m]));
              a4[m] += k + m >= lo && k + m < hi ? x : 0.f;
            }
          }
        }
      }
      w += (a4[0] + a4[1]) + (a4[2] + a4[3]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[kWbSEmpty + buf]);
        mbar_arrive(&bars[kWbEmpty + s]);
      }
    }
    if (ok && j < sq.len) p.kw[b * p.kw_sb + kh * p.kw_sh + j] += w;
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

template <int D, int RP>
cudaError_t launch_key_weights_t(const KwMaps& m, const KeyWeightsParams& p, cudaStream_t stream) {
  using L = KwSmem<D, RP>;
  auto kern = fna2_key_weights_kernel<D, RP>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed);
  if (e != cudaSuccess) return e;
  const int64_t n = static_cast<int64_t>(p.bd.T) * std::max<int64_t>(p.H, static_cast<int64_t>(p.kv.hg) * p.RP / 8);
  fna2_key_weights_prep_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const dim3 grid(p.kv.hkv, (p.bd.max_k + 2 * kBlockN - 1) / (2 * kBlockN), p.bd.B);
  kern<<<grid, kKwThreads, L::kTotal, stream>>>(m.q, m.k, m.rq, m.rk, p);
  return cudaGetLastError();
}

inline cudaError_t launch_key_weights(const KwMaps& m, const KeyWeightsParams& p, int D, cudaStream_t stream) {
  if (D == 64) return p.RP == 16 ? launch_key_weights_t<64, 16>(m, p, stream) : launch_key_weights_t<64, 32>(m, p, stream);
  return p.RP == 16 ? launch_key_weights_t<128, 16>(m, p, stream) : launch_key_weights_t<128, 32>(m, p, stream);
}

}  // namespace fna2
