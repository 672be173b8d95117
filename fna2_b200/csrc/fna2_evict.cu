// Eviction from a paged cache by accumulated attention weight.
//
// Per sequence and KV head: of its `len` keys keep min(len, budget): the first
// `sink`, the last `recent`, and of the others those of the largest weight, ties
// to the lowest index (NaN ranks below every number).  The kept keys' rows of
// K, V and of the KV head's query heads' R_k move, in order, to slots [0, kept) of
// the pages of another table, so rows are never overwritten while they are read
// and pages that several sequences share stay as they are.
//
// Two kernels.  Select: one CTA per (sequence, KV head) finds the K-th largest
// weight by a radix search over the ordered bits of the fp32 weights (11 + 11 +
// 10 bits, a shared-memory histogram per pass), then writes the kept indices in
// order, a run of keys per warp.  It is bound by instructions: 1,024 threads of one SM,
// some 60 instructions per weight in all (16,384 weights: 16 us; 30,000 clk, of which
// loading and the first histogram 6,000, each further pass 4,000, writing 9,000).  Move:
// HBM-bound, 16-byte copies of whole rows (64 heads' caches cut to 4,096 rows of D = 128,
// 4 heads of rank 16: 57 us, 5.9 TB/s read and written).
#include "fna2_paged.cuh"

namespace fna2 {

struct EvictParams {
  PagedPool kv;  // source table
  const int* lens;
  int B, G, D, max_k, budget, sink, recent;
  const float* w;
  int64_t w_sb, w_sh;
  const int* table_out;
  int64_t table_out_sb;
  int cap_out;       // slots of an output table row
  int* kept;         // [B][HKV][budget], -1 past the kept count
  int* lens_out;     // [B]
  float* w_out;      // [B][HKV][cap_out], 0 past the kept count
};

struct RowPlace {
  int sp, ss, dp, ds;  // source page (-1: none) and slot, destination page and slot
};

// Copies kept rows [r0, r1), at most ROWS of them, of (sequence b, KV head kh) with a block of THREADS threads.
template <int THREADS, int ROWS>
__device__ __forceinline__ void move_rows(const EvictParams& p, int b, int kh, int r0, int r1, const int* kept,
                                          RowPlace* s_at) {
  const int mask = (1 << p.kv.page_log2) - 1, tid = threadIdx.x, rows = min(ROWS, r1 - r0);
  if (tid < rows) {
    const int r = r0 + tid, j = kept[r];
    RowPlace a{-1, j & mask, -1, r & mask};
    if (j >= 0) {
      a.sp = __ldg(p.kv.table + b * p.kv.table_sb + (j >> p.kv.page_log2));
      a.dp = __ldg(p.table_out + b * p.table_out_sb + (r >> p.kv.page_log2));
      if (a.sp < 0 || a.sp >= p.kv.pages || a.dp < 0 || a.dp >= p.kv.pages) {
        atomicCAS(&g_device_error, 0, kStatusBadSeqEvict);
        a.sp = -1;
      }
    }
    s_at[tid] = a;
  }
  __syncthreads();
  // K and V: 2 D / 8 lanes a row, four rows in flight per lane
  constexpr int U = 4;
  const int warp = tid >> 5, lane = tid & 31, lpr = p.D / 4, rpw = 32 / lpr;
  const int sub = lane % lpr, is_v = sub >= lpr / 2, col = sub % (lpr / 2) * 8;
  const PagedRows kv = {is_v ? p.kv.v.ptr : p.kv.k.ptr, is_v ? p.kv.v.sp : p.kv.k.sp, is_v ? p.kv.v.st : p.kv.k.st,
                        is_v ? p.kv.v.sh : p.kv.k.sh};
  for (int base = warp * rpw * U; base < rows; base += THREADS / 32 * rpw * U) {
    uint4 v[U];
    __nv_bfloat16* dst[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = base + i * rpw + lane / lpr;
      dst[i] = nullptr;
      if (r < rows && s_at[r].sp >= 0) {
        const RowPlace a = s_at[r];
        v[i] = *reinterpret_cast<const uint4*>(kv.ptr + paged_off(kv, a.sp, a.ss, kh) + col);
        dst[i] = kv.ptr + paged_off(kv, a.dp, a.ds, kh) + col;
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (dst[i]) *reinterpret_cast<uint4*>(dst[i]) = v[i];
  }
  // R_k of the KV head's query heads
  const int r8 = p.kv.rank / 8, pieces = max(0, min(p.G, p.kv.hg - kh * p.G)) * r8;
  for (int base = tid; base < rows * pieces; base += THREADS * U) {
    uint4 v[U];
    __nv_bfloat16* dst[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int e = base + i * THREADS, r = e / pieces, c = e % pieces;
      dst[i] = nullptr;
      if (e < rows * pieces && s_at[r].sp >= 0) {
        const RowPlace a = s_at[r];
        const int64_t at = (kh * p.G + c / r8) * p.kv.rk.sh + c % r8 * 8;
        v[i] = *reinterpret_cast<const uint4*>(p.kv.rk.ptr + paged_off(p.kv.rk, a.sp, a.ss, 0) + at);
        dst[i] = p.kv.rk.ptr + paged_off(p.kv.rk, a.dp, a.ds, 0) + at;
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (dst[i]) *reinterpret_cast<uint4*>(dst[i]) = v[i];
  }
}

// Kept rows up to which the select kernel moves them itself.  Of 4 sequences, 4 heads that takes as long on the
// GPU as two kernels do (512 rows 8.4 us) and spares the host a launch (16.0 against 18.3 us per call); of 32
// sequences 512 rows take 14.4 against 15.8 us, 1,024 rows 21.4 against 22.9.
constexpr int kFusedBudget = 1024;
constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048;
constexpr int kHistCopies = 2;  // lanes that count the same bin at once wait for each other: even and odd ones apart

// fp32 bits in an order-preserving unsigned form; -0 equals +0, NaN is lowest.
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  const int u = __float_as_int(x + 0.f);
  return x != x ? 0u : static_cast<uint32_t>(u ^ (u >> 31 | static_cast<int>(0x80000000u)));
}

// MOVE: the block also copies rows (small budgets: one launch instead of two).  Then several blocks (z) find
// the same keys, as long as there are SMs, and each copies its share of their rows.  STAGED: the
// sequence's weights fit in shared memory and are read from there after the first pass (each pass over
// 16,384 weights in global memory took 7 us, latency of dependent loads).
template <bool MOVE, bool STAGED>
__global__ void __launch_bounds__(kSelThreads) fna2_evict_select_kernel(const EvictParams p) {
  extern __shared__ float s_w[];
  __shared__ int hist[kHistCopies][kSelBins];
  __shared__ RowPlace s_at[MOVE ? kFusedBudget : 1];
  __shared__ int s_kept[MOVE ? kFusedBudget : 1];
  __shared__ int s_warp[2][32];
  __shared__ int s_digit, s_above;
  const int kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  int len = __ldg(p.lens + b);
  if (len < 0 || len > p.max_k) {
    if (tid == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqEvict);
    len = 0;
  }
  const int keep = min(len, p.budget);
  const int old_end = max(0, len - p.recent), old_beg = min(p.sink, old_end);  // candidates [old_beg, old_end)
  const int need = keep - (len - old_end) - old_beg;                            // >= 0: sink + recent <= budget
  const float* w = p.w + b * p.w_sb + kh * p.w_sh;
  const bool all = need >= old_end - old_beg, some = !all && need > 0;
  // weights j .. j + 3 (j a multiple of 4); anything past the candidates
  auto load4 = [&](int j, float* x) {
    if (STAGED) {
      *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(s_w + j);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = j + i < old_end ? __ldg(w + j + i) : 0.f;
    }
  };
  // bit i: key j + i is a candidate below `end`
  auto candidates = [&](int j, int end) {
    if (j >= old_beg && j + 3 < end) return 15u;
    unsigned in = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) in |= static_cast<unsigned>(j + i >= old_beg && j + i < end) << i;
    return in;
  };
  int* my_hist = hist[tid % kHistCopies];
  uint32_t prefix = 0;
  int want = need;  // rank of the threshold among the candidates that share the prefix
  if (STAGED || some) {
    for (int i = tid; i < kHistCopies * kSelBins; i += kSelThreads) hist[0][i] = 0;
    __syncthreads();
  }
  if (STAGED) {
    constexpr int U = 8;  // loads in flight
    for (int j0 = tid; j0 < len; j0 += U * kSelThreads) {
      float x[U];
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = j0 + i * kSelThreads < len ? __ldg(w + j0 + i * kSelThreads) : 0.f;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int j = j0 + i * kSelThreads;
        if (j < len) {
          s_w[j] = x[i];
          if (j >= old_beg && j < old_end) atomicAdd(&my_hist[ordered_bits(x[i]) >> 21], 1);
        }
      }
    }
    __syncthreads();
  }
  if (some) {
    int shift = 32;
    for (int pass = 0; pass < 3; ++pass) {
      const int width = pass < 2 ? 11 : 10;
      const uint32_t hi_mask = pass == 0 ? 0u : 0xffffffffu << shift;
      shift -= width;
      if (!STAGED || pass > 0) {
        for (int j = (old_beg & ~3) + 4 * tid; j < old_end; j += 4 * kSelThreads) {
          alignas(16) float x[4];
          load4(j, x);
          const unsigned in = candidates(j, old_end);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t u = ordered_bits(x[i]);
            if ((u & hi_mask) == prefix && (in >> i & 1))
              atomicAdd(&my_hist[(u >> shift) & ((1u << width) - 1)], 1);
          }
        }
        __syncthreads();
      }
      // suffix counts: thread t owns bins 2t and 2t + 1
      int c0 = 0, c1 = 0;
#pragma unroll
      for (int i = 0; i < kHistCopies; ++i) {
        int2* c = reinterpret_cast<int2*>(&hist[i][2 * tid]);
        c0 += c->x, c1 += c->y;
        *c = make_int2(0, 0);  // for the next pass
      }
      const int mine = c0 + c1;
      int suf = mine;  // inclusive suffix sum within the warp
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_down_sync(0xffffffffu, suf, o);
        if (lane + o < 32) suf += v;
      }
      if (lane == 0) s_warp[0][warp] = suf;
      __syncthreads();
      const int after = __reduce_add_sync(0xffffffffu, lane > warp ? s_warp[0][lane] : 0);
      const int above1 = after + suf - mine;  // candidates in bins above 2t + 1
      const int above0 = above1 + c1;
      if (above1 < want && want <= above1 + c1) s_digit = 2 * tid + 1, s_above = above1;
      if (above0 < want && want <= above0 + c0) s_digit = 2 * tid, s_above = above0;
      __syncthreads();
      prefix |= static_cast<uint32_t>(s_digit) << shift;
      want -= s_above;
      __syncthreads();
    }
  }
  // prefix: the threshold value; want: how many candidates equal to it are kept (the lowest indices).
  if (all) prefix = 0, want = len;
  if (!all && !some) prefix = 0xffffffffu;  // above every weight
  int* kept = p.kept + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.budget;
  float* w_out = p.w_out + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.cap_out;
  const bool writes = !MOVE || blockIdx.z == 0;
  auto put = [&](int pos, int j, float x) {
    if (MOVE) s_kept[pos] = j;
    if (writes) kept[pos] = j, w_out[pos] = x;
  };
  for (int j = tid; j < old_beg; j += kSelThreads) put(j, j, STAGED ? s_w[j] : __ldg(w + j));
  for (int j = old_end + tid; j < len; j += kSelThreads) put(keep - len + j, j, STAGED ? s_w[j] : __ldg(w + j));
  // Each warp owns a run of the keys: it counts the candidates that it takes, then writes from its offset on.
  const int run = (old_end + 4 * kSelThreads - 1) / (4 * kSelThreads) * 128;
  const int beg = min(old_end, warp * run), end = min(old_end, beg + run);
  // Of keys j .. j + 3: bits of those taken for certain, and of those equal to the threshold.
  auto flags = [&](const float* x, unsigned in, unsigned* take, unsigned* tie) {
    *take = *tie = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = ordered_bits(x[i]);
      if (u > prefix) *take |= 1u << i;
      if (u == prefix) *tie |= 1u << i;
    }
    *take &= in, *tie &= in;
  };
  int takes = 0, ties = 0;
  for (int j = beg + 4 * lane; j < end; j += 128) {
    alignas(16) float x[4];
    load4(j, x);
    unsigned mt, me;
    flags(x, candidates(j, end), &mt, &me);
    takes += __popc(mt), ties += __popc(me);
  }
  takes = __reduce_add_sync(0xffffffffu, takes), ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) s_warp[0][warp] = takes, s_warp[1][warp] = ties;
  __syncthreads();
  pdl_trigger();
  int takes_before = old_beg + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[0][lane] : 0);
  int ties_before = __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[1][lane] : 0);
  for (int j0 = beg; j0 < end; j0 += 128) {
    const int j = j0 + 4 * lane;
    alignas(16) float x[4];
    unsigned mt = 0, me = 0;
    if (j < end) {
      load4(j, x);
      flags(x, candidates(j, end), &mt, &me);
    }
    // takes and ties << 16 of the lanes up to this one
    const int mine = __popc(mt) | __popc(me) << 16;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int a = takes_before + ((incl - mine) & 0xffff), e = ties_before + ((incl - mine) >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool take = mt >> i & 1, tie = me >> i & 1;
      if (take || (tie && e < want)) {
        put(a + min(e, want), j + i, x[i]);
      }
      a += take, e += tie;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    takes_before += total & 0xffff, ties_before += total >> 16;
  }
  if (writes) {
    for (int i = keep + tid; i < p.budget; i += kSelThreads) kept[i] = -1;
    for (int i = keep + tid; i < p.cap_out; i += kSelThreads) w_out[i] = 0.f;
    if (kh == 0 && tid == 0) p.lens_out[b] = keep;
  }
  if (MOVE) {
    __syncthreads();  // s_kept is written
    const int z = blockIdx.z, nz = gridDim.z;
    move_rows<kSelThreads, kFusedBudget>(p, b, kh, keep * z / nz, keep * (z + 1) / nz, s_kept, s_at);
  }
}

constexpr int kMoveThreads = 128;
constexpr int kMoveRows = 32;

__global__ void __launch_bounds__(kMoveThreads) fna2_evict_move_kernel(const EvictParams p) {
  __shared__ RowPlace s_at[kMoveRows];
  pdl_wait();
  const int b = blockIdx.z, kh = blockIdx.y, r0 = blockIdx.x * kMoveRows;
  move_rows<kMoveThreads, kMoveRows>(p, b, kh, r0, p.budget, p.kept + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.budget,
                                     s_at);
}

// Weights that fit in shared memory beside the histograms and the kept rows' places.
constexpr int kStagedKeys = 40 * 1024;

template <bool MOVE>
cudaError_t launch_evict_select(const EvictParams& p, cudaStream_t stream) {
  const dim3 heads(p.kv.hkv, p.B, MOVE ? std::max(1, std::min(8, kSms / (p.kv.hkv * p.B))) : 1);
  if (p.max_k <= kStagedKeys) {
    auto kern = fna2_evict_select_kernel<MOVE, true>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed, kStagedKeys * 4);
    if (e != cudaSuccess) return e;
    return launch_dependent(kern, heads, kSelThreads, (p.max_k + 3) / 4 * 16, stream, p);
  }
  return launch_dependent(fna2_evict_select_kernel<MOVE, false>, heads, kSelThreads, 0, stream, p);
}

inline cudaError_t launch_evict(const EvictParams& p, cudaStream_t stream) {
  if (p.budget <= kFusedBudget) return launch_evict_select<true>(p, stream);
  const cudaError_t e = launch_evict_select<false>(p, stream);
  if (e != cudaSuccess) return e;
  return launch_dependent(fna2_evict_move_kernel, dim3((p.budget + kMoveRows - 1) / kMoveRows, p.kv.hkv, p.B),
                          kMoveThreads, 0, stream, p);
}

}  // namespace fna2
