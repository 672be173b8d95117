// Shared pieces of the paged-cache kernels: the pool of pages, the sequence
// bounds of a call, and the split of one sequence's keys over CTAs.
#pragma once

#include <atomic>

#include "fna2_kernels.cuh"
#include "ptx.cuh"

namespace fna2 {

constexpr int kSms = 148;  // of a B200

// Site codes recorded in g_device_error (read by fna2_device_status).
constexpr int kStatusBadSeqAppend = 631;  // append: bad length / offsets, or a page id outside the pool
constexpr int kStatusBadSeqPaged = 641;   // attention, key weights: bad length or offsets, or a page id outside the pool
constexpr int kStatusBadSeqEvict = 651;   // eviction: bad length, or a page id outside the pool

struct PagedRows {  // one tensor of the pool: element (page, slot, head, column), column stride 1
  __nv_bfloat16* ptr;
  int64_t sp, st, sh;
};

struct PagedPool {
  int pages, page_log2;  // pages in the pool, log2 of the slots per page
  int hkv, hg, rank;
  PagedRows k, v, rk;
  const int* table;  // [B, max_pages] page ids
  int64_t table_sb;
  int max_pages;
};

// First element of key j's row of head `head` (page id already looked up).
__device__ __forceinline__ int64_t paged_off(const PagedRows& r, int page_id, int slot, int head) {
  return page_id * r.sp + slot * r.st + head * r.sh;
}

// Attention and key weights: a page id that a key needs, outside the pool, is recorded; its keys read as zeros
// (bounds checks here, out-of-range tensor-map coordinates there).
__device__ __forceinline__ void check_page(const PagedPool& kv, int page) {
  if (page < 0 || page >= kv.pages) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
}

struct PagedSeq {
  int q0, n;   // first packed token, number of new tokens
  int len;     // cached keys, the new tokens' among them
  bool ok;
};

// The bounds that a call's grids and workspaces were sized by.
struct PagedBounds {
  int B, T, max_q, max_k;
  const int* cu;
  const int* lens;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedBounds& p, int b) {
  PagedSeq s;
  s.q0 = __ldg(p.cu + b);
  const int e = __ldg(p.cu + b + 1);
  s.len = __ldg(p.lens + b);
  s.ok = s.q0 >= 0 && e >= s.q0 && e <= p.T && e - s.q0 <= p.max_q && s.len >= 0 && s.len <= p.max_k;
  s.n = s.ok ? e - s.q0 : 0;
  if (!s.ok) s.len = 0;
  return s;
}

// hi + lo = f * x to 2^-17 relative, both bf16, for 8 bf16 values x (see fna2_paged.cu).
__device__ __forceinline__ void split_bias(const uint4& x, float f, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  const uint32_t xx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&xx[i]));
    const float a = v.x * f, b = v.y * f;
    hi[i] = pack_bf16(a, b);
    const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&hi[i]));
    lo[i] = pack_bf16(a - y.x, b - y.y);
  }
}

// Sequence of packed token t (cu ascending): the last b with cu[b] <= t, found
// by the whole warp, 32 probes a round.  -1 when t lies outside [cu[0], cu[B]).
__device__ __forceinline__ int warp_seq_of(const int* cu, int B, int64_t t, int lane) {
  if (t < __ldg(cu) || t >= __ldg(cu + B)) return -1;
  int lo = 0, hi = B;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int idx = min(lo + lane * step, hi);
    const bool le = idx < hi && __ldg(cu + idx) <= t;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    lo += max(0, 31 - __clz(static_cast<int>(m))) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

// Programmatic dependent launch: a kernel launched with launch_dependent may start while the kernel
// before it runs its last CTAs, once all of those have called pdl_trigger or exited; pdl_wait returns
// when that kernel is complete and its writes are visible.  Every kernel launched this way calls
// pdl_wait in a thread of every block, so work after it in the stream is ordered as usual.  The first
// kernel of a call waits before it does anything else, its trigger included: the ones after it may read
// the call's inputs without a wait of their own.  That launch saves about a microsecond of a small call
// even then (append of 48 tokens 14.2 -> 13.5 us, attention of 16 drafts 30.8 -> 29.1).
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... P, class... A>
cudaError_t launch_dependent(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &a;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kern, static_cast<P>(args)...);
}

// Lets a kernel use all of the dynamic shared memory (or `bytes` of it), once per device (`done`: a
// bit per device; the call costs about a microsecond, a small kernel takes five).
inline cudaError_t allow_smem(const void* kern, std::atomic<uint64_t>& done, int bytes = kMaxDynamicSmem) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace fna2
