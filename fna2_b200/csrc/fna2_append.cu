// New tokens into a paged cache: per-head RMSNorm and rotary embedding of q and
// k at each sequence's own position, and k, v, r_k written into their pages.
//
//   n = x * rsqrt(mean(x^2) + eps) * w
//   y = n * cos(pos f) + rotate_half(n) * sin(pos f),  rotate_half(n) = [-n2, n1]
// with pos = positions[b] + i for new token i of sequence b, the arithmetic and
// the roundings of fna2_qk_prep_kernel (so a key that is appended equals the
// one the packed training path forms for the same position, bit for bit).
//
// HBM- or launch-bound: every input row is read once and written once.  One CTA
// per token: the sequence search, the page lookup and the D/2 sincosf are done
// once and serve all heads of the token.  128 threads and 10 CTAs per SM: the time is
// latency (loads 8.6, barriers 3.4 of 17.8 clk per instruction at 256 threads and 4
// CTAs), so residency counts; 8,555 tokens of 16 + 16 heads, D = 128, rank 32, fp32 in:
// 68.7 us at 256 threads x 4 CTAs, 62.6 at 256 x 5, 57.5 at 128 x 10 (5.7 TB/s).
#include "fna2_paged.cuh"

namespace fna2 {

struct AppendRows {
  const void* ptr;
  int64_t ts, hs;  // token, head strides (elements)
};

struct AppendParams {
  PagedPool kv;
  int T, B, H;
  int w_bf16, rope_bf16;
  AppendRows q, k, v, rk;
  __nv_bfloat16* qo;
  int64_t qo_ts, qo_hs;
  const int* cu;
  const int* lens;       // slots in use before the call
  const int* positions;  // position of each sequence's first new token, or NULL (= lens)
  const void* qw;
  const void* kw;
  float eps;
  const float* inv_freq;
};

constexpr int kAppendThreads = 128;

// 8 consecutive values from global memory.
template <int EB>
__device__ __forceinline__ void ldg8(const void* base, int64_t off, float (&x)[8]) {
  if (EB == 2) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + off));
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ww[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&y)[8]) {
  return make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
}

template <int D, int EB>
__global__ void __launch_bounds__(kAppendThreads, 10) fna2_append_kernel(const AppendParams p) {
  constexpr int LPR = D / 16, RPW = 32 / LPR, NW = kAppendThreads / 32;  // lanes per row, rows per warp
  __shared__ float s_cos[D / 2], s_sin[D / 2];
  __shared__ int s_seq[4];  // page id (-1: skip the token), slot, position
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane % LPR;
  pdl_wait();
  pdl_trigger();
  if (warp == 0) {
    const int b = warp_seq_of(p.cu, p.B, t, lane);
    int page = -1, slot = 0, pos = 0;
    if (b >= 0) {
      const int first = __ldg(p.cu + b), n = __ldg(p.cu + b + 1) - first, len = __ldg(p.lens + b);
      const int64_t j = static_cast<int64_t>(len) + (t - first);
      const int64_t cap = static_cast<int64_t>(p.kv.max_pages) << p.kv.page_log2;
      pos = (p.positions ? __ldg(p.positions + b) : len) + (t - first);
      if (len >= 0 && static_cast<int64_t>(len) + n <= cap) {
        page = __ldg(p.kv.table + b * p.kv.table_sb + (j >> p.kv.page_log2));
        slot = static_cast<int>(j & ((1 << p.kv.page_log2) - 1));
      }
      if (page < 0 || page >= p.kv.pages) {
        page = -1;
        if (lane == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqAppend);
      }
    }
    if (lane == 0) s_seq[0] = page, s_seq[1] = slot, s_seq[2] = pos;
  }
  __syncthreads();
  const int page = s_seq[0], slot = s_seq[1];
  if (page < 0) return;
  const bool rope = p.inv_freq != nullptr, norm = p.qw != nullptr;
  if (rope && tid < D / 2) {
    const float tf = static_cast<float>(s_seq[2]), f = __ldg(p.inv_freq + tid);
    const float ang = p.rope_bf16 ? bf16_round(bf16_round(tf) * bf16_round(f)) : tf * f;
    float s, c;
    sincosf(ang, &s, &c);
    s_cos[tid] = p.rope_bf16 ? bf16_round(c) : c;
    s_sin[tid] = p.rope_bf16 ? bf16_round(s) : s;
  }
  __syncthreads();

  // q and k rows: lane `sub` of a row holds columns [8 sub, +8) of both halves
  const int rows = p.H + p.kv.hkv;
  for (int r0 = warp * RPW; r0 < rows; r0 += NW * RPW) {
    const int r = r0 + lane / LPR;
    const bool live = r < rows, isq = r < p.H;
    float x1[8], x2[8];
    if (live) {
      const void* src = isq ? p.q.ptr : p.k.ptr;
      const int64_t off = isq ? t * p.q.ts + r * p.q.hs : t * p.k.ts + (r - p.H) * p.k.hs;
      ldg8<EB>(src, off + 8 * sub, x1);
      ldg8<EB>(src, off + D / 2 + 8 * sub, x2);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x1[i] = x2[i] = 0.f;
    }
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x1[i], x1[i], fmaf(x2[i], x2[i], ss));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss * (1.f / D) + p.eps);
      const void* w = isq ? p.qw : p.kw;
      float w1[8], w2[8];
      if (p.w_bf16)
        ldg8<2>(w, 8 * sub, w1), ldg8<2>(w, D / 2 + 8 * sub, w2);
      else
        ldg8<4>(w, 8 * sub, w1), ldg8<4>(w, D / 2 + 8 * sub, w2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x1[i] = x1[i] * inv * w1[i];
        x2[i] = x2[i] * inv * w2[i];
      }
    }
    uint4 y1, y2;
    if (rope) {
      float c[8], s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s_cos[8 * sub + i], s[i] = s_sin[8 * sub + i];
      if (p.rope_bf16) {
        rope_bf16_packed(x1, x2, c, s, y1, y2);
      } else {
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[i] = __fadd_rn(__fmul_rn(x1[i], c[i]), -__fmul_rn(x2[i], s[i]));
          b[i] = __fadd_rn(__fmul_rn(x2[i], c[i]), __fmul_rn(x1[i], s[i]));
        }
        y1 = pack8(a), y2 = pack8(b);
      }
    } else {
      y1 = pack8(x1), y2 = pack8(x2);
    }
    if (live) {
      __nv_bfloat16* dst = isq ? p.qo + t * p.qo_ts + r * p.qo_hs : p.kv.k.ptr + paged_off(p.kv.k, page, slot, r - p.H);
      *reinterpret_cast<uint4*>(dst + 8 * sub) = y1;
      *reinterpret_cast<uint4*>(dst + D / 2 + 8 * sub) = y2;
    }
  }
  // v and r_k rows: 8 columns a thread
  const int v_pieces = p.kv.hkv * (D / 8), r8 = p.kv.rank / 8, pieces = v_pieces + p.kv.hg * r8;
  for (int e = tid; e < pieces; e += kAppendThreads) {
    float x[8];
    if (e < v_pieces) {
      const int h = e / (D / 8), c = e % (D / 8) * 8;
      ldg8<EB>(p.v.ptr, t * p.v.ts + h * p.v.hs + c, x);
      *reinterpret_cast<uint4*>(p.kv.v.ptr + paged_off(p.kv.v, page, slot, h) + c) = pack8(x);
    } else {
      const int h = (e - v_pieces) / r8, c = (e - v_pieces) % r8 * 8;
      ldg8<EB>(p.rk.ptr, t * p.rk.ts + h * p.rk.hs + c, x);
      *reinterpret_cast<uint4*>(p.kv.rk.ptr + paged_off(p.kv.rk, page, slot, h) + c) = pack8(x);
    }
  }
}

inline cudaError_t launch_append(const AppendParams& p, int D, int elem_bytes, cudaStream_t stream) {
  auto kern = D == 128 ? (elem_bytes == 2 ? fna2_append_kernel<128, 2> : fna2_append_kernel<128, 4>)
                       : (elem_bytes == 2 ? fna2_append_kernel<64, 2> : fna2_append_kernel<64, 4>);
  return launch_dependent(kern, p.T, kAppendThreads, 0, stream, p);
}

}  // namespace fna2
