// Attention weight that each cached key received:
//   w[b, kh, j] += sum over query heads h of KV head kh and new tokens i that
//                  see key j of exp(S[h,i,j] - LSE[h,i])
// with S and LSE as in the paged attention.  The logits are recomputed from
// [q | R~_q hi, lo] and [k | r_k]; a thread sums the weights of its own keys, so
// no two threads add to the same key and the result does not depend on timing.
//
// Simple form: one CTA per 64 keys of a (sequence, KV head), 16 keys a warp; the
// query rows pass through shared memory 16 at a time (mma.sync m16n8k16).
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
};

constexpr int kKwThreads = 128;
constexpr int kKwKeys = 64;

__host__ __device__ inline int kw_k_stride(int D, int ng, int RP) { return (D + ng * RP) * 2 + 16; }
__host__ __device__ inline int kw_a_stride(int D, int RP) { return (D + 2 * RP) * 2 + 16; }

template <int D>
__global__ void __launch_bounds__(kKwThreads) fna2_key_weights_kernel(const KeyWeightsParams p) {
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ float s_lse[16];
  const int kh = blockIdx.y, b = blockIdx.z, j_base = blockIdx.x * kKwKeys;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedSeq sq = paged_seq(p.bd, b);
  if (!sq.ok && tid == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
  if (j_base >= sq.len || sq.n == 0) return;
  const int past = sq.len - sq.n;
  const int ng = max(0, min(p.G, p.kv.hg - kh * p.G)), ngs = min(p.G, p.kv.hg);
  const int k_stride = kw_k_stride(D, ngs, p.RP), a_stride = kw_a_stride(D, p.RP);
  uint8_t* sk = dsm;
  uint8_t* sa = dsm + kKwKeys * k_stride;
  const int pieces = D / 8 + ng * (p.RP / 8);
  for (int e = tid; e < kKwKeys * pieces; e += kKwThreads) {
    const int r = e / pieces, c = e % pieces, j = j_base + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (j < sq.len) {
      const int page = __ldg(p.kv.table + b * p.kv.table_sb + (j >> p.kv.page_log2));
      const int slot = j & ((1 << p.kv.page_log2) - 1);
      if (page >= 0 && page < p.kv.pages) {
        if (c < D / 8) {
          v = *reinterpret_cast<const uint4*>(p.kv.k.ptr + paged_off(p.kv.k, page, slot, kh) + c * 8);
        } else {
          const int g = (c - D / 8) / (p.RP / 8), col = (c - D / 8) % (p.RP / 8) * 8;
          if (col < p.kv.rank)
            v = *reinterpret_cast<const uint4*>(p.kv.rk.ptr + paged_off(p.kv.rk, page, slot, kh * p.G + g) + col);
        }
      }
    }
    *reinterpret_cast<uint4*>(sk + r * k_stride + c * 16) = v;
  }
  const int g = lane >> 2, t = lane & 3;
  const int jw = j_base + warp * 16;
  const int kk[4] = {jw + 2 * t, jw + 2 * t + 1, jw + 8 + 2 * t, jw + 9 + 2 * t};
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t a_addr = smem_u32(sa) + ((lane & 7) + ((lane >> 3) & 1) * 8) * a_stride + (lane >> 4) * 16;
  const uint32_t k_addr =
      smem_u32(sk) + (warp * 16 + (lane & 7) + (lane >> 4) * 8) * k_stride + ((lane >> 3) & 1) * 16;
  const int i_first = p.causal ? max(0, j_base - past) / 16 * 16 : 0;  // earlier tokens see none of these keys
  for (int gg = 0; gg < p.G; ++gg) {
    const int h = kh * p.G + gg;
    const bool graph = h < p.kv.hg;
    for (int i0 = i_first; i0 < sq.n; i0 += 16) {
      __syncthreads();
      const int ap = D / 8 + (graph ? p.RP / 8 : 0);
      for (int e = tid; e < 16 * ap; e += kKwThreads) {
        const int r = e / ap, c = e % ap, i = i0 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < D / 8) {
          if (i < sq.n) v = *reinterpret_cast<const uint4*>(p.q + (sq.q0 + i) * p.q_st + h * p.q_sh + c * 8);
          *reinterpret_cast<uint4*>(sa + r * a_stride + c * 16) = v;
        } else {
          const int col = (c - D / 8) * 8;
          uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
          if (i < sq.n && col < p.kv.rank) {
            v = *reinterpret_cast<const uint4*>(p.rq + (sq.q0 + i) * p.rq_st + h * p.rq_sh + col);
            split_bias(v, __ldg(p.gs + h) / p.scale, hi, lo);
          }
          *reinterpret_cast<uint4*>(sa + r * a_stride + c * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(sa + r * a_stride + (c + p.RP / 8) * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      if (tid < 16) {
        const float v = i0 + tid < sq.n ? __ldg(p.lse + h * p.lse_sh + sq.q0 + i0 + tid) : -INFINITY;
        s_lse[tid] = v == -INFINITY ? INFINITY : v * kLog2e;  // a row without weight adds 0
      }
      __syncthreads();
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[4], kb[4];
        ldsm_x4(a, a_addr + ks * 32);
        ldsm_x4(kb, k_addr + ks * 32);
        mma_bf16(s0, a, kb[0], kb[1]);
        mma_bf16(s1, a, kb[2], kb[3]);
      }
      if (graph)
        for (int ks = 0; ks < p.RP / 16; ++ks) {
          uint32_t a[4], kb[4];
          ldsm_x4(kb, k_addr + (D + gg * p.RP) * 2 + ks * 32);
          ldsm_x4(a, a_addr + D * 2 + ks * 32);
          mma_bf16(s0, a, kb[0], kb[1]);
          mma_bf16(s1, a, kb[2], kb[3]);
          ldsm_x4(a, a_addr + (D + p.RP) * 2 + ks * 32);
          mma_bf16(s0, a, kb[0], kb[1]);
          mma_bf16(s1, a, kb[2], kb[3]);
        }
      const float xa[4] = {s0[0], s0[1], s1[0], s1[1]}, xb[4] = {s0[2], s0[3], s1[2], s1[3]};
      const int ia = i0 + g, ib = ia + 8;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (ia < sq.n && (!p.causal || kk[c] <= past + ia)) w[c] += exp2f(fmaf(xa[c], p.scale_log2, -s_lse[g]));
        if (ib < sq.n && (!p.causal || kk[c] <= past + ib)) w[c] += exp2f(fmaf(xb[c], p.scale_log2, -s_lse[g + 8]));
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) w[c] += __shfl_xor_sync(0xffffffffu, w[c], o);
  if (g == 0)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (kk[c] < sq.len) p.kw[b * p.kw_sb + kh * p.kw_sh + kk[c]] += w[c];
}

inline int key_weights_smem(int D, int ng, int RP) { return kKwKeys * kw_k_stride(D, ng, RP) + 16 * kw_a_stride(D, RP); }

template <int D>
cudaError_t launch_key_weights_t(const KeyWeightsParams& p, cudaStream_t stream) {
  auto kern = fna2_key_weights_kernel<D>;
  const int smem = key_weights_smem(D, std::min(p.G, p.kv.hg), p.RP);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kern<<<dim3((p.bd.max_k + kKwKeys - 1) / kKwKeys, p.kv.hkv, p.bd.B), kKwThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

inline cudaError_t launch_key_weights(const KeyWeightsParams& p, int D, cudaStream_t stream) {
  return D == 128 ? launch_key_weights_t<128>(p, stream) : launch_key_weights_t<64>(p, stream);
}

}  // namespace fna2
