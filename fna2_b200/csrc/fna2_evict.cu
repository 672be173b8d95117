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
// order with a block-wide scan.  Move: HBM-bound, 16-byte copies of whole rows.
#include "fna2_paged.cuh"

namespace fna2 {

struct EvictParams {
  PagedPool kv;  // source table
  const int* lens;
  int B, G, max_k, budget, sink, recent;
  const float* w;
  int64_t w_sb, w_sh;
  const int* table_out;
  int64_t table_out_sb;
  int cap_out;       // slots of an output table row
  int* kept;         // [B][HKV][budget], -1 past the kept count
  int* lens_out;     // [B]
  float* w_out;      // [B][HKV][cap_out], 0 past the kept count
};

constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048;

// fp32 bits in an order-preserving unsigned form; -0 equals +0, NaN is lowest.
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelThreads) fna2_evict_select_kernel(const EvictParams p) {
  __shared__ int hist[kSelBins];
  __shared__ int s_warp[2][32];
  __shared__ int s_digit, s_above;
  const int kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int len = __ldg(p.lens + b);
  if (len < 0 || len > p.max_k) {
    if (tid == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqEvict);
    len = 0;
  }
  const int keep = min(len, p.budget);
  const int old_end = max(0, len - p.recent), old_beg = min(p.sink, old_end);  // candidates [old_beg, old_end)
  const int need = keep - (len - old_end) - old_beg;                            // >= 0: sink + recent <= budget
  const float* w = p.w + b * p.w_sb + kh * p.w_sh;
  uint32_t prefix = 0;
  int want = need;  // rank of the threshold among the candidates that share the prefix
  const bool all = need >= old_end - old_beg;
  if (!all && need > 0) {
    int shift = 32;
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      const uint32_t hi_mask = pass == 0 ? 0u : 0xffffffffu << shift;
      shift -= bits;
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j = old_beg + tid; j < old_end; j += kSelThreads) {
        const uint32_t u = ordered_bits(__ldg(w + j));
        if ((u & hi_mask) == prefix) atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      // suffix counts: thread t owns bins 2t and 2t + 1
      const int c1 = hist[2 * tid + 1], c0 = hist[2 * tid], mine = c0 + c1;
      int suf = mine;  // inclusive suffix sum within the warp
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_down_sync(0xffffffffu, suf, o);
        if (lane + o < 32) suf += v;
      }
      if (lane == 0) s_warp[0][warp] = suf;
      __syncthreads();
      int after = 0;
      for (int i = warp + 1; i < 32; ++i) after += s_warp[0][i];
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
  // prefix: the threshold value; want: how many candidates equal to it are kept (the lowest indices)
  int* kept = p.kept + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.budget;
  float* w_out = p.w_out + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.cap_out;
  int base = 0, ties = 0;
  for (int j0 = 0; j0 < len; j0 += kSelThreads) {
    const int j = j0 + tid;
    bool take = false, tie = false;
    float x = 0.f;
    if (j < len) {
      x = __ldg(w + j);
      const uint32_t u = ordered_bits(x);
      const bool cand = j >= old_beg && j < old_end;
      take = !cand || all || (need > 0 && u > prefix);
      tie = cand && !all && need > 0 && u == prefix;
    }
    const unsigned mt = __ballot_sync(0xffffffffu, take), me = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) s_warp[0][warp] = __popc(mt), s_warp[1][warp] = __popc(me);
    __syncthreads();
    int take_before = 0, tie_before = 0, take_all = 0, tie_all = 0;
    for (int i = 0; i < 32; ++i) {
      const int a = s_warp[0][i], c = s_warp[1][i];
      if (i < warp) take_before += a, tie_before += c;
      take_all += a, tie_all += c;
    }
    const unsigned lt = (1u << lane) - 1;
    const int my_ties = ties + tie_before + __popc(me & lt);
    const int pos = base + take_before + __popc(mt & lt) + min(my_ties, want) - min(ties, want);
    if (take || (tie && my_ties < want)) {
      kept[pos] = j;
      w_out[pos] = x;
    }
    base += take_all + min(ties + tie_all, want) - min(ties, want);
    ties += tie_all;
    __syncthreads();
  }
  for (int i = keep + tid; i < p.budget; i += kSelThreads) kept[i] = -1;
  for (int i = keep + tid; i < p.cap_out; i += kSelThreads) w_out[i] = 0.f;
  if (kh == 0 && tid == 0) p.lens_out[b] = keep;
}

constexpr int kMoveThreads = 128;
constexpr int kMoveRows = 32;

__global__ void __launch_bounds__(kMoveThreads) fna2_evict_move_kernel(const EvictParams p, int D) {
  __shared__ int s_src[kMoveRows][2], s_dst[kMoveRows][2];  // page, slot
  const int kh = blockIdx.y, b = blockIdx.z, r0 = blockIdx.x * kMoveRows, tid = threadIdx.x;
  const int* kept = p.kept + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.budget;
  const int mask = (1 << p.kv.page_log2) - 1;
  if (tid < kMoveRows) {
    const int r = r0 + tid, j = r < p.budget ? kept[r] : -1;
    int sp = -1, dp = -1;
    if (j >= 0) {
      sp = __ldg(p.kv.table + b * p.kv.table_sb + (j >> p.kv.page_log2));
      dp = __ldg(p.table_out + b * p.table_out_sb + (r >> p.kv.page_log2));
      if (sp < 0 || sp >= p.kv.pages || dp < 0 || dp >= p.kv.pages) {
        atomicCAS(&g_device_error, 0, kStatusBadSeqEvict);
        sp = -1;
      }
    }
    s_src[tid][0] = sp, s_src[tid][1] = j & mask;
    s_dst[tid][0] = dp, s_dst[tid][1] = r & mask;
  }
  __syncthreads();
  const int ppr = D / 8, r8 = p.kv.rank / 8, ng = max(0, min(p.G, p.kv.hg - kh * p.G));
  const int pieces = 2 * ppr + ng * r8;
  for (int e = tid; e < kMoveRows * pieces; e += kMoveThreads) {
    const int r = e / pieces, c = e % pieces;
    const int sp = s_src[r][0], ss = s_src[r][1], dp = s_dst[r][0], ds = s_dst[r][1];
    if (sp < 0) continue;
    if (c < 2 * ppr) {
      const PagedRows& t = c < ppr ? p.kv.k : p.kv.v;
      const int col = c % ppr * 8;
      *reinterpret_cast<uint4*>(t.ptr + paged_off(t, dp, ds, kh) + col) =
          *reinterpret_cast<const uint4*>(t.ptr + paged_off(t, sp, ss, kh) + col);
    } else {
      const int h = kh * p.G + (c - 2 * ppr) / r8, col = (c - 2 * ppr) % r8 * 8;
      *reinterpret_cast<uint4*>(p.kv.rk.ptr + paged_off(p.kv.rk, dp, ds, h) + col) =
          *reinterpret_cast<const uint4*>(p.kv.rk.ptr + paged_off(p.kv.rk, sp, ss, h) + col);
    }
  }
}

inline cudaError_t launch_evict(const EvictParams& p, int D, cudaStream_t stream) {
  fna2_evict_select_kernel<<<dim3(p.kv.hkv, p.B), kSelThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  fna2_evict_move_kernel<<<dim3((p.budget + kMoveRows - 1) / kMoveRows, p.kv.hkv, p.B), kMoveThreads, 0, stream>>>(p, D);
  return cudaGetLastError();
}

}  // namespace fna2
