// Attention weight that each cached key received:
//   w[b, kh, j] += sum over query heads h of KV head kh and new tokens i that
//                  see key j of exp(S[h,i,j] - LSE[h,i])
// with S and LSE as in the paged attention (fna2_paged.cu).
//
// On the tensor cores, the transposed scores
//   S^T - LSE/scale = [K | R_k | R_k | 1] [Q | R~_q hi | R~_q lo | -LSE/scale]^T
// put a key on every TMEM lane, so the thread that owns a key sums its weights over
// the columns in a register: no reduction within a warp, no atomics on the result, which
// does not depend on timing.  The LSE is one more K slice, three bf16 terms that hold its
// 24 bits, so that a column costs the sum warps one exp2, half a multiplication and half an
// addition (packed pairs).  A small kernel first writes the R~_q hi / lo and LSE columns.
// Persistent CTAs, one per SM, work on units of 128 columns:
//   fna2_key_weights_kernel         key-stationary: an item is a pair of 128-key tiles
//     of a (sequence, KV head), drawn from a counter (items differ: early keys are seen
//     by more queries), a unit 128 queries of one head; every Q tile serves both.
//     Warpgroup i sums key tile i % 2 of every second unit.
//   fna2_key_weights_window_kernel  query-stationary, when no sequence has more than
//     64 queries: a CTA takes an equal run of all key tiles, the queries of up to four
//     heads stay in shared memory while K and R_k stream (streaming Q past each key tile
//     instead took 128 KB per tile from L2 where this takes 48: 64 queries, 4 caches of up
//     to 16,000 keys, 32 heads 82 against 37 us, 8 heads 38 / 26); a unit is two heads side
//     by side (one N = 128 product with K, then each head's R_k against its half).
//     Warpgroup i sums head i % 2 of every second unit.
// Warps 0-15: sums (four warps per scheduler: with two, waits between units showed); 16:
// TMA (K and R_k page by page, as in fna2_paged_many.cu); 17: TMEM allocation, MMA issue;
// 18: waits for warp 17 (a wait by the warp that issued MMAs returns only when its own MMAs
// have drained; a named barrier does not); 19: adds the warpgroups' sums of a key tile and
// updates the weights (a load per key that the sum warps would wait for).
// Bound: the products and their hand-offs.  The 26 MMAs of a unit (two key tiles) take 1,860
// clk, 1,660 of them at the tensor pipe's rate; with waits and hand-offs a unit takes 2,450
// clk key-stationary (4,095 queries and keys, 16 heads, D = 128, rank 32:
// 55.5 us, 780 TFLOP/s), 2,400 per key tile and four heads query-stationary, where a tile's 48 KB also need
// 2,900 clk from a freed stage to a full one and two stages fit (64 queries, 4 caches of up to
// 16,000 keys, 8 KV heads of 4, rank 16: 37 us, 3.5 TB/s).  exp2 (2,048 clk of the same) is
// not what bounds it: a polynomial on the FMA pipe for a quarter of them halved the sums' time
// and changed neither kernel's.  Nor did two issuing warps, or two loading ones.
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
  __nv_bfloat16* rq2;  // workspace: [T][H][2 RP + 16]: R~_q hi, lo (graph heads), -LSE/scale as three terms
  int* next;           // workspace: item counter, set to ctas (whose first items are their own index) by the prep kernel
  int ctas;
  int64_t clear;       // > 0: the weights are set, not added to; values of each row of kw to write
};

// If weights are set: 0 for the keys that no query sees.  R~_q = gs/scale * R_q as hi + lo, columns [rank, RP) zero, and -LSE/scale = l1 + l2 + l3 (a row
// without weight: -1e38, whose weights are 0).
__global__ void __launch_bounds__(256) fna2_key_weights_prep_kernel(const KeyWeightsParams p) {
  pdl_wait();
  pdl_trigger();
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e == 0) *p.next = p.ctas;
  for (int64_t row = p.clear > 0 ? blockIdx.x : INT64_MAX; row < static_cast<int64_t>(p.bd.B) * p.kv.hkv; row += gridDim.x) {
    const int b = static_cast<int>(row / p.kv.hkv), kh = static_cast<int>(row % p.kv.hkv);
    const PagedSeq s = paged_seq(p.bd, b);
    float* dst = p.kw + b * p.kw_sb + kh * p.kw_sh;
    for (int64_t x = (s.n > 0 ? s.len / 4 : 0) + threadIdx.x; x < p.clear / 4; x += 256)
      reinterpret_cast<float4*>(dst)[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int r8 = p.RP / 8, per = r8 + 1;  // pieces of a row: R_q's, then the LSE's
  if (e >= static_cast<int64_t>(p.bd.T) * p.H * per) return;
  const int x = static_cast<int>(e % per), h = static_cast<int>(e / per % p.H);
  const int64_t t = e / per / p.H;
  __nv_bfloat16* dst = p.rq2 + (t * p.H + h) * (2 * p.RP + 16);
  if (x == r8) {
    const float lse = p.lse[h * p.lse_sh + t];
    const float c = lse == -INFINITY ? -1e38f : -lse / p.scale;
    const float l1 = __bfloat162float(__float2bfloat16_rn(c)), l2 = __bfloat162float(__float2bfloat16_rn(c - l1));
    *reinterpret_cast<uint4*>(dst + 2 * p.RP) = make_uint4(pack_bf16(l1, l2), pack_bf16(c - l1 - l2, 0.f), 0, 0);
    *reinterpret_cast<uint4*>(dst + 2 * p.RP + 8) = make_uint4(0, 0, 0, 0);
  } else if (h < p.kv.hg) {
    uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
    if (8 * x < p.kv.rank)
      split_bias(*reinterpret_cast<const uint4*>(p.rq + t * p.rq_st + h * p.rq_sh + 8 * x), __ldg(p.gs + h) / p.scale,
                 hi, lo);
    *reinterpret_cast<uint4*>(dst + 8 * x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(dst + p.RP + 8 * x) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

constexpr int kKwThreads = 640;
constexpr int kKwProducer = 16, kKwIssuer = 17, kKwWaiter = 18;  // warps after the sums; then the one that stores

template <int D, int RP>
struct KwSmem {
  static constexpr int kTile = 128 * D * 2;            // K tile, Q of a unit
  static constexpr int kRTile = 128 * RP * 2;          // R_k of a key tile, R~_q hi or lo of a unit
  static constexpr int kChunk = 128 * 128;             // 64 columns of a 128-row tile
  static constexpr int kLTile = 128 * 32;              // the LSE's K slice of a unit, the ones against it
  static constexpr int oK = 0;                         // key tiles 0, 1
  static constexpr int oStage = oK + 2 * kTile;        // 2 x [Q | R~_q hi, lo | LSE]
  static constexpr int sQ = 0, sRq = kTile, sL = sRq + 2 * kRTile;
  static constexpr int kStage = sL + kLTile;
  static constexpr int oRk = oStage + 2 * kStage;      // 2 x R_k of key tiles 0, 1 and the unit's head
  static constexpr int oOne = oRk + 2 * 2 * kRTile;
  static constexpr int oPart = oOne + kLTile;          // sums of warpgroup i of key tile i % 2
  static constexpr int oBar = oPart + 4 * 512;
  static constexpr int oMisc = oBar + 32 * 8;
  static constexpr int oItem = oMisc + 16;
  static constexpr int kUsed = oItem + 64;
  static constexpr int kTotal = kUsed + 1024;
  static_assert(kTotal <= kMaxDynamicSmem, "shared memory budget");
  static_assert(kStage % 1024 == 0, "swizzle atoms stay aligned");
};

enum KwBar {
  kWbKFull = 0,    // K and the item's description
  kWbKEmpty = 1,   // its MMAs are done, every warp has read its description (1 + 17 arrivals)
  kWbPFull = 2,    // the item's sums (16 arrivals)
  kWbPEmpty = 3,
  kWbFull = 4,     // +stage: the unit's operands
  kWbEmpty = 6,    // +stage: MMAs that read it are done
  kWbSFull = 8,    // +2 tile + buffer
  kWbSEmpty = 12,  // +2 tile + buffer (one arrival per warp)
};

struct KwItem {
  int b, kh, k0, len, n, q0, u0, per_head, n_units;  // n_units < 0: no more items; u0: first query tile that sees keys
};

// Item `idx`: (`keys` keys, KV head) of the sequences in packing order, the KV heads of the same keys
// together, early keys (which the most queries see) first.  Called by a whole warp.
__device__ __forceinline__ KwItem kw_item(const KeyWeightsParams& p, int idx, int keys, int lane) {
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
      if (s.n > 0) cnt = (s.len + keys - 1) / keys * p.kv.hkv;
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
      it.k0 = local / p.kv.hkv * keys;
      it.len = __shfl_sync(0xffffffffu, s.len, src);
      it.n = __shfl_sync(0xffffffffu, s.n, src);
      it.q0 = __shfl_sync(0xffffffffu, s.q0, src);
      const int n_qt = (it.n + kBlockM - 1) / kBlockM;
      it.u0 = p.causal ? min(n_qt, max(0, it.k0 - (it.len - it.n)) / kBlockM) : 0;  // earlier tokens see none of these keys
      it.per_head = n_qt - it.u0;
      it.n_units = it.per_head * p.G;
      return it;
    }
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  return it;
}

// The ones against the LSE's three terms: 128 rows of 16 columns, of which 0-2, 32-byte swizzled.
__device__ __forceinline__ void kw_write_ones(uint8_t* dst) {
  for (int e = threadIdx.x; e < 256; e += kKwThreads)
    *reinterpret_cast<uint4*>(dst + e * 16) =
        (e & 1) == ((e >> 3) & 1) ? make_uint4(0x3f803f80u, 0x00003f80u, 0, 0) : make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
}

// Sum over columns [lo, hi) of this thread's lane of 2^(sl2 S), 16 at a time; `hi` is the warp's, `lo` the
// thread's.  (Masks cost 5 instructions per column: `cut` says whether some thread of the tile has lo > 0,
// and the chunk that hi ends in needs them; two loops, so that the common one stays unrolled.)
template <int QT>
__device__ __forceinline__ float kw_sum(uint32_t t_addr, float2 sl2, int lo, int hi, bool cut) {
  float2 a[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t r[2][16];
  tmem_ld16(t_addr, r[0]);
  if (!cut && hi >= QT) {
#pragma unroll
    for (int c = 0; c < QT / 16; ++c) {
      uint32_t* x = r[c & 1];
      tmem_ld_wait16(x);
      if (c + 1 < QT / 16) tmem_ld16(t_addr + 16 * (c + 1), r[(c + 1) & 1]);
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        const float2 y = __fmul2_rn(f32x2(x[k], x[k + 1]), sl2);
        a[k / 2 & 1] = __fadd2_rn(a[k / 2 & 1], make_float2(ex2(y.x), ex2(y.y)));
      }
    }
  } else {
#pragma unroll 1
    for (int c0 = 0; c0 < QT && c0 < hi; c0 += 32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = c0 + 16 * i;
        uint32_t* x = r[i];
        tmem_ld_wait16(x);
        if (c + 16 < QT && c + 16 < hi) tmem_ld16(t_addr + c + 16, r[i ^ 1]);
        if (c >= hi) continue;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          const float2 y = __fmul2_rn(f32x2(x[k], x[k + 1]), sl2);
          float2 e = make_float2(ex2(y.x), ex2(y.y));
          e.x = c + k >= lo && c + k < hi ? e.x : 0.f;
          e.y = c + k + 1 >= lo && c + k + 1 < hi ? e.y : 0.f;
          a[k / 2 & 1] = __fadd2_rn(a[k / 2 & 1], e);
        }
      }
    }
  }
  return (a[0].x + a[0].y) + (a[1].x + a[1].y);
}

template <int D, int RP>
__global__ void __launch_bounds__(kKwThreads, 1)
    fna2_key_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmRq, const __grid_constant__ CUtensorMap tmRk,
                            const __grid_constant__ CUtensorMap tmL, const KeyWeightsParams p) {
  using L = KwSmem<D, RP>;
  constexpr int QT = 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::oMisc + 4);
  volatile KwItem* items = reinterpret_cast<volatile KwItem*>(smem + L::oItem);
  const int warp = warp_id(), lane = lane_id(), tid = threadIdx.x;

  if (tid == 0) {
    mbar_init(&bars[kWbKFull], 1);
    mbar_init(&bars[kWbKEmpty], 18);
    mbar_init(&bars[kWbPFull], 16);
    mbar_init(&bars[kWbPEmpty], 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kWbFull + s], 1);
      mbar_init(&bars[kWbEmpty + s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars[kWbSFull + s], 1);
      mbar_init(&bars[kWbSEmpty + s], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  kw_write_ones(smem + L::oOne);
  if (warp == kKwIssuer) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kKwProducer) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
    }
    const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
    const int bk = min(1 << lg, kBlockN);  // rows of a box; lane l owns box l of the key tiles (at most 16)
    const int tile = lane * bk / kBlockN, row = lane * bk % kBlockN;
    // Items are drawn and their pages looked up while earlier units wait for room.
    auto draw = [&]() {
      int idx = 0;
      if (lane == 0) idx = atomicAdd(p.next, 1);
      return kw_item(p, __shfl_sync(0xffffffffu, idx, 0), 2 * kBlockN, lane);
    };
    auto page_of = [&](const KwItem& it) {
      const int key = it.k0 + lane * bk;
      if (it.n_units < 0 || lane * bk >= 2 * kBlockN || key >= it.len) return -1;
      const int page = __ldg(p.kv.table + it.b * p.kv.table_sb + (key >> lg));
      check_page(p.kv, page);
      return page;
    };
    KwItem it = kw_item(p, blockIdx.x, 2 * kBlockN, lane), next = it;
    int page = page_of(it), next_page = -1;
    int gu = 0, rs = 1;  // units so far, R_k slot
    for (int n = 0;; ++n) {
      const bool free = n < 1 || mbar_wait(&bars[kWbKEmpty], (n - 1) & 1, abort_flag, 120);
      if (!__all_sync(0xffffffffu, free)) break;
      const int key = it.k0 + lane * bk;
      const bool mine = it.n_units >= 0 && lane * bk < 2 * kBlockN && key < it.len;
      const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) {  // (the arrival also publishes the description)
        volatile KwItem* d = items;
        d->b = it.b, d->kh = it.kh, d->k0 = it.k0, d->len = it.len, d->n = it.n, d->u0 = it.u0;
        d->per_head = it.per_head, d->n_units = it.n_units;
        mbar_expect_tx(&bars[kWbKFull], boxes * bk * D * 2);
      }
      __syncwarp();
      if (it.n_units < 0) break;
      if (mine) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + L::oK + tile * L::kTile + c * L::kChunk + row * 128, &tmK,
                      &bars[kWbKFull], c * 64, key & mask, it.kh, page);
      }
      __syncwarp();
      if (n == 0) pdl_wait();  // the prep kernel writes nothing of what was read so far
      auto fetch = [&]() {
        next = draw();
        next_page = page_of(next);
      };
      if (it.n_units == 0) fetch();
      bool ok = true;
      for (int u = 0; u < it.n_units; ++u, ++gu) {
        const int s = gu & 1;
        const int h = it.kh * p.G + u / it.per_head, tok = it.q0 + (it.u0 + u % it.per_head) * QT;
        const bool graph = h < p.kv.hg;
        uint8_t* st = smem + L::oStage + s * L::kStage;
        // R_k: unless this unit's head is the last one's.  The slot's former readers are done: the unit before
        // the last one is, and at least one unit has used the other slot since.
        const bool fresh = u % it.per_head == 0;
        if (fresh) rs ^= 1;
        const bool room = gu < 2 || mbar_wait(&bars[kWbEmpty + s], ((gu >> 1) - 1) & 1, abort_flag, 121);
        ok = __all_sync(0xffffffffu, room);
        if (!ok) break;
        if (lane == 0)
          mbar_expect_tx(&bars[kWbFull + s],
                         QT * (D + 16 + (graph ? 2 * RP : 0)) * 2 + (fresh && graph ? boxes * bk * RP * 2 : 0));
        __syncwarp();
        // lanes 16, 17: Q chunks; 24, 25: R~_q hi, lo; 28: LSE
        const int x = lane - 16, y = lane - 24;
        const bool is_q = x >= 0 && x < D / 64, is_r = graph && y >= 0 && y < 2;
        if (is_q || is_r || lane == 28)
          tma_load_4d(st + (is_q ? L::sQ + x * L::kChunk : is_r ? L::sRq + y * L::kRTile : L::sL),
                      is_q ? &tmQ : is_r ? &tmRq : &tmL, &bars[kWbFull + s], is_q ? x * 64 : is_r ? y * RP : 2 * RP, tok, h,
                      0);
        if (mine && fresh && graph)
          tma_load_4d(smem + L::oRk + (2 * rs + tile) * L::kRTile + row * RP * 2, &tmRk, &bars[kWbFull + s], 0, key & mask,
                      h, page);
        __syncwarp();
        if (u == max(0, it.n_units - 2)) fetch();  // not earlier: who draws early gets work before it is free
      }
      if (!ok) break;
      it = next, page = next_page;
    }
  } else if (warp == kKwIssuer || warp == kKwWaiter) {
    // ------------------------------------------------------------ MMA issuer and its waiter
    constexpr uint32_t idesc = make_idesc_bf16(kBlockN, 128, 0, 0);
    constexpr uint32_t r_layout = RP == 16 ? kSwizzle32B : kSwizzle64B;
    constexpr uint32_t r_sbo = 8 * RP * 2;
    const bool issuer = warp == kKwIssuer;
    // operand descriptors at their first stage; others differ in the address field only (bytes / 16)
    const uint32_t s0 = smem_u32(smem);
    const uint64_t dK0 = make_sdesc(s0 + L::oK, 16, 1024, kSwizzle128B);
    const uint64_t dQ0 = make_sdesc(s0 + L::oStage + L::sQ, 16, 1024, kSwizzle128B);
    const uint64_t dOne = make_sdesc(s0 + L::oOne, 16, 256, kSwizzle32B);
    const uint64_t dL0 = make_sdesc(s0 + L::oStage + L::sL, 16, 256, kSwizzle32B);
    const uint64_t dRk0 = make_sdesc(s0 + L::oRk, 16, r_sbo, r_layout);
    const uint64_t dRq0 = make_sdesc(s0 + L::oStage + L::sRq, 16, r_sbo, r_layout);
    int gu = 0, rs = 1, used[2] = {};
    bool ok = true;
    for (int n = 0; ok; ++n) {
      ok = issuer || mbar_wait(&bars[kWbKFull], n & 1, abort_flag, 221);
      ok = pair_rendezvous(1, ok);
      if (!ok) break;
      const int n_units = items[0].n_units, per_head = items[0].per_head, kh = items[0].kh;
      const int tiles = items[0].k0 + kBlockN < items[0].len ? 2 : 1;
      if (n_units < 0) break;
      for (int u = 0; ok && u < n_units; ++u, ++gu) {
        const int s = gu & 1;
        const bool graph = kh * p.G + u / per_head < p.kv.hg;
        if (u % per_head == 0) rs ^= 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= tiles) continue;
          const int buf = 2 * i + used[i] % 2;
          if (!issuer) {
            ok = used[i] < 2 || mbar_wait(&bars[kWbSEmpty + buf], (used[i] / 2 - 1) & 1, abort_flag, 223);
            if (ok && i == 0) ok = mbar_wait(&bars[kWbFull + s], (gu >> 1) & 1, abort_flag, 222);
          }
          ++used[i];
          ok = pair_rendezvous(1, ok);
          if (!ok) break;
          if (issuer) tc_fence_after();
          if (issuer && elect_one()) {
            const uint32_t tS = tmem + 128 * buf;
            const uint64_t dK = dK0 + (i * L::kTile >> 4), dQ = dQ0 + (s * L::kStage >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * L::kChunk + (kk & 3) * 32) >> 4;
              mma_ss(tS, dK + off, dQ + off, idesc, kk > 0);
            }
            mma_ss(tS, dOne, dL0 + (s * L::kStage >> 4), idesc, 1);
            if (graph) {
              const uint64_t dRk = dRk0 + ((2 * rs + i) * L::kRTile >> 4), dRq = dRq0 + (s * L::kStage >> 4);
#pragma unroll
              for (int kk = 0; kk < RP / 16; ++kk) {
                mma_ss(tS, dRk + kk * 2, dRq + kk * 2, idesc, 1);
                mma_ss(tS, dRk + kk * 2, dRq + (L::kRTile >> 4) + kk * 2, idesc, 1);
              }
            }
            mma_commit(&bars[kWbSFull + buf]);
            if (i == tiles - 1) mma_commit(&bars[kWbEmpty + s]);
          }
        }
        __syncwarp();
      }
      if (ok && issuer && elect_one()) mma_commit(&bars[kWbKEmpty]);
      __syncwarp();
    }
  } else if (warp < kKwProducer) {
    // ------------------------------------------------------------ sums: warpgroup i, key tile i % 2, every second unit
    const int wi = warp >> 2 & 1, half = warp >> 3;
    const int buf = 2 * wi + half;
    const uint32_t at = tmem + 128 * buf + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float* part = reinterpret_cast<float*>(smem + L::oPart) + (warp >> 2) * 128 + (tid & 127);
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    int used = 0;  // units of this key tile so far
    bool ok = true;
    for (int n = 0; ok; ++n) {
      if (!mbar_wait(&bars[kWbKFull], n & 1, abort_flag, 320)) break;
      const int n_units = items[0].n_units, per_head = items[0].per_head, u0 = items[0].u0, nq = items[0].n;
      const int len = items[0].len, tile0 = items[0].k0 + wi * kBlockN, j = tile0 + (tid & 127), past = len - nq;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kWbKEmpty]);
      if (n_units < 0) break;
      float w = 0.f;
      if (tile0 < len) {  // this key tile has keys
        for (int u = (half ^ used) & 1; u < n_units; u += 2) {
          if (!(ok = mbar_wait(&bars[kWbSFull + buf], ((used + u) >> 1) & 1, abort_flag, 322))) break;
          tc_fence_after();
          const int i0 = (u0 + u % per_head) * QT;
          // columns [first, nq - i0) belong to queries that see the key; the score of another sequence's
          // query is never read into a sum
          const int first = p.causal ? j - past - i0 : 0;
          w += kw_sum<QT>(at, sl2, first, nq - i0, p.causal && tile0 + kBlockN - 1 > past + i0);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[kWbSEmpty + buf]);
        }
        used += n_units;
      }
      if (!ok || (n > 0 && !mbar_wait(&bars[kWbPEmpty], (n - 1) & 1, abort_flag, 323))) break;
      *part = w;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kWbPFull]);
    }
  } else {
    // ------------------------------------------------------------ adds the warpgroups' sums and stores
    const float* part = reinterpret_cast<const float*>(smem + L::oPart) + lane;
    pdl_wait();  // the prep kernel may write up to three weights past those it leaves out
    for (int n = 0;; ++n) {
      if (!mbar_wait(&bars[kWbKFull], n & 1, abort_flag, 330)) break;
      const int left = items[0].len - items[0].k0 - lane, n_units = items[0].n_units;
      float* dst = p.kw + items[0].b * p.kw_sb + items[0].kh * p.kw_sh + items[0].k0 + lane;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kWbKEmpty]);
      if (n_units < 0) break;
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = 32 * k < left && p.clear == 0 ? dst[32 * k] : 0.f;
      if (!mbar_wait(&bars[kWbPFull], n & 1, abort_flag, 331)) break;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (32 * k < left) dst[32 * k] = w[k] + (part[32 * k] + part[256 + 32 * k]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kWbPEmpty]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kKwIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// query-stationary form: at most 64 queries per sequence
// ---------------------------------------------------------------------------
template <int D, int RP>
struct KwwSmem {
  static constexpr int kPairs = D == 128 && RP == 32 ? 1 : 2;  // head pairs whose queries stay
  static constexpr int kHeads = 2 * kPairs;
  static constexpr int kTile = 128 * D * 2;                    // K tile, Q of a head pair
  static constexpr int kRTile = 128 * RP * 2;                  // R_k of a head, R~_q hi or lo of a head pair
  static constexpr int kChunk = 128 * 128;
  static constexpr int kLTile = 128 * 32;
  static constexpr int sRq = kTile, sL = sRq + 2 * kRTile, kPair = sL + kLTile;  // [Q | R~_q hi, lo | LSE] of a pair
  static constexpr int oQ = 0;
  static constexpr int oK = oQ + kPairs * kPair;               // 2 x [K | R_k of each head]
  static constexpr int kStage = kTile + kHeads * kRTile;
  static constexpr int oOne = oK + 2 * kStage;
  static constexpr int oPart = oOne + kLTile;                  // 2 x sums of four warpgroups
  static constexpr int oBar = oPart + 2 * 4 * 512;
  static constexpr int oMisc = oBar + 32 * 8;
  static constexpr int oItem = oMisc + 16;
  static constexpr int kUsed = oItem + 64;
  static constexpr int kTotal = kUsed + 1024;
  static_assert(kTotal <= kMaxDynamicSmem, "shared memory budget");
  static_assert(kPair % 1024 == 0 && kStage % 1024 == 0, "swizzle atoms stay aligned");
};

enum KwwBar {
  kVbQFull = 0,    // the queries and the step's description
  kVbQEmpty = 1,   // the step's MMAs are done, every warp has read its description (1 + 17 arrivals)
  kVbFull = 2,     // +stage: K and R_k of a key tile
  kVbEmpty = 4,    // +stage
  kVbSFull = 6,    // +buffer
  kVbSEmpty = 10,  // +buffer (8 arrivals)
  kVbPFull = 14,   // +tile parity: the key tile's sums (16 arrivals)
  kVbPEmpty = 16,  // +tile parity
};

// A step: `tiles` key tiles from key k0 on against heads [h0, h0 + heads) of one KV head.
struct KwwStep {
  int b, kh, k0, len, n, tiles, h0, heads;  // tiles < 0: no more steps
};

// Up to `most` key tiles of one KV head from position `at` on, in the order: sequences, blocks of key tiles, KV
// heads, key tiles (the KV heads of the same keys at about the same time: a token's heads lie together).  Blocks of
// a sequence are equal, of `block` key tiles or a few more, so that a run meets few of them.
// Called by a whole warp.
struct KwwRun {
  int b, kh, k0, len, n, q0, tiles;
};

__device__ __forceinline__ KwwRun kww_run(const KeyWeightsParams& p, int at, int most, int block, int lane) {
  KwwRun it{};
  int carry = 0;
  for (int base = 0; base < p.bd.B; base += 32) {
    const int b = base + lane;
    PagedSeq s{0, 0, 0, false};
    int cnt = 0;
    if (b < p.bd.B) {
      s = paged_seq(p.bd, b);
      if (s.n > 0) cnt = (s.len + kBlockN - 1) / kBlockN * p.kv.hkv;
    }
    int incl = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, at < carry + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int local = at - carry - (__shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, cnt, src));
      it.b = base + src;
      it.len = __shfl_sync(0xffffffffu, s.len, src);
      it.n = __shfl_sync(0xffffffffu, s.n, src);
      it.q0 = __shfl_sync(0xffffffffu, s.q0, src);
      const int tiles = (it.len + kBlockN - 1) / kBlockN, blocks = max(1, tiles / block);
      const int blk = ((local / p.kv.hkv + 1) * static_cast<int64_t>(blocks) - 1) / tiles;
      const int first = static_cast<int64_t>(blk) * tiles / blocks, in = local - first * p.kv.hkv;
      const int size = static_cast<int>((blk + 1ll) * tiles / blocks) - first;
      it.kh = in / size;
      it.k0 = (first + in % size) * kBlockN;
      it.tiles = min(most, size - in % size);
      return it;
    }
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  return it;
}

template <int D, int RP>
__global__ void __launch_bounds__(kKwThreads, 1)
    fna2_key_weights_window_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                   const __grid_constant__ CUtensorMap tmRq, const __grid_constant__ CUtensorMap tmRk,
                                   const __grid_constant__ CUtensorMap tmL, const KeyWeightsParams p) {
  using L = KwwSmem<D, RP>;
  constexpr int QT = 64, NB = 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::oMisc + 4);
  volatile KwwStep* step = reinterpret_cast<volatile KwwStep*>(smem + L::oItem);
  const int warp = warp_id(), lane = lane_id(), tid = threadIdx.x;

  if (tid == 0) {
    mbar_init(&bars[kVbQFull], 1);
    mbar_init(&bars[kVbQEmpty], 18);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kVbFull + s], 1);
      mbar_init(&bars[kVbEmpty + s], 1);
      mbar_init(&bars[kVbPFull + s], 16);
      mbar_init(&bars[kVbPEmpty + s], 1);
    }
    for (int s = 0; s < NB; ++s) {
      mbar_init(&bars[kVbSFull + s], 1);
      mbar_init(&bars[kVbSEmpty + s], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  kw_write_ones(smem + L::oOne);
  if (warp == kKwIssuer) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kKwProducer) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
    }
    const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
    const int bk = min(1 << lg, kBlockN), row = lane * bk;  // lane l owns box l of a key tile (at most 8)
    int total = 0;  // key tiles of all KV heads
    for (int base = 0; base < p.bd.B; base += 32) {
      int cnt = 0;
      if (base + lane < p.bd.B) {
        const PagedSeq s = paged_seq(p.bd, base + lane);
        if (!s.ok) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
        if (s.n > 0) cnt = (s.len + kBlockN - 1) / kBlockN * p.kv.hkv;
      }
      total += __reduce_add_sync(0xffffffffu, cnt);
    }
    const int C = static_cast<int>(gridDim.x), c = static_cast<int>(blockIdx.x), run = total / C, more = total % C;
    int at = c * run + min(c, more);
    const int end = at + run + (c < more);
    int gt = 0;  // key tiles so far
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const bool last = at == end;
      KwwRun it;
      if (!last) it = kww_run(p, at, end - at, run + (more > 0), lane);
      const int tiles = last ? -1 : it.tiles;
      for (int g0 = 0; ok && g0 < p.G; g0 += L::kHeads) {
        const int h0 = it.kh * p.G + g0, nh = min(L::kHeads, p.G - g0), ng = max(0, min(nh, p.kv.hg - h0));
        auto load = [&](int t) {  // key tile t
          const int s = gt & 1, key = it.k0 + t * kBlockN + row;
          const bool mine = row < kBlockN && key < it.len;
          const int page = mine ? __ldg(p.kv.table + it.b * p.kv.table_sb + (key >> lg)) : 0;
          if (mine) check_page(p.kv, page);
          const bool room = gt < 2 || mbar_wait(&bars[kVbEmpty + s], ((gt >> 1) - 1) & 1, abort_flag, 126);
          if (!(ok = __all_sync(0xffffffffu, room))) return;
          const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
          if (lane == 0) mbar_expect_tx(&bars[kVbFull + s], boxes * bk * (D + ng * RP) * 2);
          __syncwarp();
          uint8_t* st = smem + L::oK + s * L::kStage;
          if (mine) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(st + c * L::kChunk + row * 128, &tmK, &bars[kVbFull + s], c * 64, key & mask, it.kh, page);
            for (int hh = 0; hh < ng; ++hh)
              tma_load_4d(st + L::kTile + hh * L::kRTile + row * RP * 2, &tmRk, &bars[kVbFull + s], 0, key & mask, h0 + hh,
                          page);
          }
          __syncwarp();
          ++gt;
        };
        if (!last) load(0);  // before the queries, which wait for the last step's MMAs
        if (!ok) break;
        const bool free = n == 0 || mbar_wait(&bars[kVbQEmpty], (n - 1) & 1, abort_flag, 125);
        if (!(ok = __all_sync(0xffffffffu, free))) break;
        if (lane == 0) {  // (the arrival also publishes the description)
          step->b = it.b, step->kh = it.kh, step->k0 = it.k0, step->len = it.len, step->n = it.n, step->tiles = tiles;
          step->h0 = h0, step->heads = nh;
          mbar_expect_tx(&bars[kVbQFull], last ? 0 : QT * (nh * (D + 16) + ng * 2 * RP) * 2);
        }
        __syncwarp();
        if (last) break;
        if (n == 0) pdl_wait();  // the prep kernel writes nothing of what was read so far
        // lane 8 g + x of head g: x = 0, 1: Q chunks; 2, 3: R~_q hi, lo; 4: LSE
        const int g = lane / 8, x = lane % 8;
        if (g < nh && (x < D / 64 || x == 4 || (x / 2 == 1 && g < ng))) {
          uint8_t* dst = smem + L::oQ + g / 2 * L::kPair +
                         (x < D / 64 ? x * L::kChunk + g % 2 * QT * 128
                          : x == 4   ? L::sL + g % 2 * QT * 32
                                     : L::sRq + (x - 2) * L::kRTile + g % 2 * QT * RP * 2);
          tma_load_4d(dst, x < D / 64 ? &tmQ : x == 4 ? &tmL : &tmRq, &bars[kVbQFull],
                      x < D / 64 ? x * 64 : x == 4 ? 2 * RP : (x - 2) * RP, it.q0, h0 + g, 0);
        }
        __syncwarp();
        for (int t = 1; ok && t < tiles; ++t) load(t);
        if (g0 + L::kHeads < p.G) ++n;
      }
      if (last) break;
      at += it.tiles;
    }
  } else if (warp == kKwIssuer || warp == kKwWaiter) {
    // ------------------------------------------------------------ MMA issuer and its waiter
    constexpr uint32_t idesc = make_idesc_bf16(kBlockN, 128, 0, 0), idesc_r = make_idesc_bf16(kBlockN, QT, 0, 0);
    constexpr uint32_t r_layout = RP == 16 ? kSwizzle32B : kSwizzle64B;
    constexpr uint32_t r_sbo = 8 * RP * 2;
    const bool issuer = warp == kKwIssuer;
    // operand descriptors at their first place; others differ in the address field only (bytes / 16)
    const uint32_t s0 = smem_u32(smem);
    const uint64_t dK0 = make_sdesc(s0 + L::oK, 16, 1024, kSwizzle128B);
    const uint64_t dQ0 = make_sdesc(s0 + L::oQ, 16, 1024, kSwizzle128B);
    const uint64_t dOne = make_sdesc(s0 + L::oOne, 16, 256, kSwizzle32B);
    const uint64_t dL0 = make_sdesc(s0 + L::oQ + L::sL, 16, 256, kSwizzle32B);
    const uint64_t dRk0 = make_sdesc(s0 + L::oK + L::kTile, 16, r_sbo, r_layout);
    const uint64_t dRq0 = make_sdesc(s0 + L::oQ + L::sRq, 16, r_sbo, r_layout);
    int gt = 0, used = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      ok = issuer || mbar_wait(&bars[kVbQFull], n & 1, abort_flag, 225);
      ok = pair_rendezvous(1, ok);
      if (!ok) break;
      const int tiles = step->tiles, h0 = step->h0, heads = step->heads;
      if (tiles < 0) break;
      for (int t = 0; ok && t < tiles; ++t, ++gt) {
        const int s = gt & 1;
        const int units = (heads + 1) / 2;
        if (!issuer) {
          for (int v = used; ok && v < used + units; ++v)
            ok = v < NB || mbar_wait(&bars[kVbSEmpty + v % NB], (v / NB - 1) & 1, abort_flag, 227);
          if (ok) ok = mbar_wait(&bars[kVbFull + s], (gt >> 1) & 1, abort_flag, 226);
        }
        ok = pair_rendezvous(1, ok);
        if (!ok) break;
        if (issuer) tc_fence_after();
#pragma unroll
        for (int u = 0; u < L::kPairs; ++u) {
          if (2 * u >= heads) continue;
          const int buf = used++ % NB;
          if (issuer && elect_one()) {
            const uint32_t tS = tmem + 128 * buf;
            const uint64_t dK = dK0 + (s * L::kStage >> 4), dQ = dQ0 + (u * L::kPair >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * L::kChunk + (kk & 3) * 32) >> 4;
              mma_ss(tS, dK + off, dQ + off, idesc, kk > 0);
            }
            mma_ss(tS, dOne, dL0 + (u * L::kPair >> 4), idesc, 1);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              if (2 * u + g >= heads || h0 + 2 * u + g >= p.kv.hg) continue;
              const uint64_t dRk = dRk0 + ((s * L::kStage + (2 * u + g) * L::kRTile) >> 4);
              const uint64_t dRq = dRq0 + ((u * L::kPair + g * QT * RP * 2) >> 4);
#pragma unroll
              for (int kk = 0; kk < RP / 16; ++kk) {
                mma_ss(tS + g * QT, dRk + kk * 2, dRq + kk * 2, idesc_r, 1);
                mma_ss(tS + g * QT, dRk + kk * 2, dRq + (L::kRTile >> 4) + kk * 2, idesc_r, 1);
              }
            }
            mma_commit(&bars[kVbSFull + buf]);
            if (2 * u + 2 >= heads) mma_commit(&bars[kVbEmpty + s]);
          }
        }
        __syncwarp();
      }
      if (ok && issuer && elect_one()) mma_commit(&bars[kVbQEmpty]);
      __syncwarp();
    }
  } else if (warp < kKwProducer) {
    // ------------------------------------------------------------ sums: warpgroup i, head i % 2 of every second unit
    const int wi = warp >> 2 & 1, half = warp >> 3;
    const uint32_t t_lane = tmem + QT * wi + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float* part = reinterpret_cast<float*>(smem + L::oPart) + (warp >> 2) * 128 + (tid & 127);
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    int used = 0, gt = 0;  // units and key tiles so far
    bool ok = true;
    for (int n = 0; ok; ++n) {
      if (!mbar_wait(&bars[kVbQFull], n & 1, abort_flag, 325)) break;
      const int tiles = step->tiles, heads = step->heads, nq = step->n, past = step->len - nq, k0 = step->k0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kVbQEmpty]);
      if (tiles < 0) break;
      for (int t = 0; ok && t < tiles; ++t, ++gt) {
        const int tile0 = k0 + t * kBlockN, first = p.causal ? tile0 + (tid & 127) - past : 0;
        float w = 0.f;
        for (int u = 0; 2 * u < heads; ++u, ++used) {
          if ((used & 1) != half) continue;
          const int buf = used % NB;
          if (!(ok = mbar_wait(&bars[kVbSFull + buf], (used / NB) & 1, abort_flag, 326))) break;
          tc_fence_after();
          // columns [first, nq) belong to queries that see the key; the score of another sequence's query
          // or of a head that the pair lacks is never read into a sum
          if (2 * u + wi < heads)
            w += kw_sum<QT>(t_lane + 128 * buf, sl2, first, nq, p.causal && tile0 + kBlockN - 1 > past);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[kVbSEmpty + buf]);
        }
        if (!ok || (gt >= 2 && !(ok = mbar_wait(&bars[kVbPEmpty + (gt & 1)], ((gt >> 1) - 1) & 1, abort_flag, 327)))) break;
        part[(gt & 1) * 512] = w;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kVbPFull + (gt & 1)]);
      }
    }
  } else {
    // ------------------------------------------------------------ adds the warpgroups' sums and stores
    const float* part = reinterpret_cast<const float*>(smem + L::oPart) + lane;
    int gt = 0;
    bool ok = true;
    pdl_wait();  // the prep kernel may write up to three weights past those it leaves out
    for (int n = 0; ok; ++n) {
      if (!mbar_wait(&bars[kVbQFull], n & 1, abort_flag, 335)) break;
      const int tiles = step->tiles;
      int left = step->len - step->k0 - lane;
      const bool set = p.clear > 0 && step->h0 == step->kh * p.G;  // the KV head's first query heads
      float* dst = p.kw + step->b * p.kw_sb + step->kh * p.kw_sh + step->k0 + lane;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kVbQEmpty]);
      if (tiles < 0) break;
      for (int t = 0; t < tiles; ++t, ++gt, left -= kBlockN, dst += kBlockN) {
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = 32 * k < left && !set ? dst[32 * k] : 0.f;
        if (!(ok = mbar_wait(&bars[kVbPFull + (gt & 1)], (gt >> 1) & 1, abort_flag, 336))) break;
        const float* x = part + (gt & 1) * 512;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (32 * k < left) dst[32 * k] = w[k] + ((x[32 * k] + x[128 + 32 * k]) + (x[256 + 32 * k] + x[384 + 32 * k]));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kVbPEmpty + (gt & 1)]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kKwIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct KwMaps {
  CUtensorMap q, k, rq, rk, l;
};

// Queries per unit: which of the two kernels runs.
inline int kw_query_tile(const KeyWeightsParams& p) { return p.bd.max_q <= 64 ? 64 : 128; }

inline cudaError_t launch_key_weights_prep(const KeyWeightsParams& p, cudaStream_t stream) {
  const int64_t n = static_cast<int64_t>(p.bd.T) * p.H * (p.RP / 8 + 1);
  const int64_t rows = p.clear > 0 ? static_cast<int64_t>(p.bd.B) * p.kv.hkv : 0;
  const int64_t blocks = std::max<int64_t>((n + 255) / 256, std::min<int64_t>(std::max<int64_t>(rows, 1), 4 * kSms));
  return launch_dependent(fna2_key_weights_prep_kernel, static_cast<unsigned>(blocks), 256, 0, stream, p);
}

template <int D, int RP>
cudaError_t launch_key_weights_t(const KwMaps& m, KeyWeightsParams& p, cudaStream_t stream) {
  const bool window = kw_query_tile(p) == 64;
  auto kern = window ? fna2_key_weights_window_kernel<D, RP> : fna2_key_weights_kernel<D, RP>;
  static std::atomic<uint64_t> allowed[2];
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed[window]);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (p.bd.max_k + kBlockN - 1) / kBlockN, seqs = static_cast<int64_t>(p.bd.B) * p.kv.hkv;
  p.ctas = static_cast<int>(std::min<int64_t>(seqs * (window ? tiles : (tiles + 1) / 2), kSms));
  e = launch_key_weights_prep(p, stream);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, static_cast<unsigned>(p.ctas), kKwThreads,
                          window ? KwwSmem<D, RP>::kTotal : KwSmem<D, RP>::kTotal, stream, m.q, m.k, m.rq, m.rk, m.l, p);
}

inline cudaError_t launch_key_weights(const KwMaps& m, KeyWeightsParams& p, int D, cudaStream_t stream) {
  if (D == 64) return p.RP == 16 ? launch_key_weights_t<64, 16>(m, p, stream) : launch_key_weights_t<64, 32>(m, p, stream);
  return p.RP == 16 ? launch_key_weights_t<128, 16>(m, p, stream) : launch_key_weights_t<128, 32>(m, p, stream);
}

}  // namespace fna2
