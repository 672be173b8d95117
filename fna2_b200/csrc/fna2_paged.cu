// Attention of new tokens over a paged cache, with the relational bias.
//
// Sequence b holds `len` cached keys (its n new tokens' own keys are the last
// n of them) in pages of a pool.  New token i, query head h, key j:
//   S = scale <q_i,h, k_j> + gs[h] <r_q,i,h, r_k[j,h]>     (h <  H_G)
//   S = scale <q_i,h, k_j>                                 (h >= H_G)
//   j is seen iff j < len and (not causal or j <= len - n + i)
//   O = acc / (l + 1e-6), LSE = m + log(l + 1e-6); a row that sees no key gets
//   O = 0 and LSE = -inf
// i.e. the last n query rows of the prefill op over the whole sequence.
//
// The factor gs/scale is folded into r_q as in the prefill kernels, but as a sum
// of two bf16 numbers, hi = bf16(f r_q) and lo = bf16(f r_q - hi) (2^-17
// relative): the LSE and the attention weights are fp32 results, and one bf16
// rounding of the bias would show in them (2^-9 of the bias).  P is rounded to
// bf16 for P V (the output is bf16); the row sums use the unrounded P.
//
// One CTA serves (sequence, KV head, block of 16 RW query rows, key split).  A
// query row is (query head of the KV group, new token), head-major, so that the
// 16 rows of a warp span few heads.  4 warps: RW row blocks x 4/RW key groups; a
// key group streams its own 16-key tiles through a ring in shared memory that its
// RW warps read together (mma.sync m16n8k16, fp32 accumulation, online softmax
// in registers).  16 keys never cross a page, so a tile is one TMA box per 64
// columns of K and V and one per head of R_k, issued by as many lanes; 128-byte
// (R_k: 32- or 64-byte) swizzled rows give conflict-free ldmatrix reads.  (With one
// cp.async per 16 bytes the address arithmetic was 3/4 of the 820 instructions a
// tile took, and the kernel was bound by their issue at 5.1 TB/s.)
// Bound: HBM; each cached key is read once per row block.
#include "fna2_paged.cuh"

namespace fna2 {

struct PagedAttnParams {
  PagedPool kv;
  PagedBounds bd;
  int H, G;       // query heads, query heads per KV head
  int RP;         // rank rounded up to 16 or 32
  int causal;
  float scale, scale_log2;
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const __nv_bfloat16* rq;
  int64_t rq_st, rq_sh;
  const float* gs;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  float* lse;  // [H][lse_sh], or NULL
  int64_t lse_sh;
  int chunk, ns;      // keys per split, splits per sequence at most
  float* ws_acc;      // [(t * H + h) * ns + split][D]: unnormalised output of a split
  float2* ws_ml;      // [(t * H + h) * ns + split]: its row max (log2 domain) and sum
  float* logits;      // key weights: [((b * HKV + kh) * max_q * G + row)][logit_sr] log2-domain logits, or NULL
  int64_t logit_sr;
  float* kw;          // key weights, added to: [b * kw_sb + kh * kw_sh + j]
  int64_t kw_sb, kw_sh;
  int row_blocks, ng_max, nh_max, stages;
  // Sequences of more than few_rows query rows (new tokens x query heads of a KV head) go to
  // fna2_paged_many_kernel, the others to fna2_paged_few_kernel; a call launches those it may need.
  int few_rows;
  int chunk_many, many_items;  // keys per split there, upper bound on its (query tile pair, split) items
};

// Splits of a sequence that hold keys.
__device__ __forceinline__ int paged_splits(const PagedAttnParams& p, const PagedSeq& s) {
  const int chunk = s.n * p.G > p.few_rows ? p.chunk_many : p.chunk;
  return max(1, (s.len + chunk - 1) / chunk);
}

constexpr int kFewThreads = 128;
constexpr int kFewKeys = 16;  // keys per tile

// Shared-memory geometry (host and device agree on it): [A of the RW row blocks | K and V ring of
// the key groups | R_k ring | barriers]; ng: graph heads of a block's rows, nh: heads that the 16
// rows of one warp span.
struct FewSmem {
  int a_stride, kv_stage, r_head, r_stage, o_kv, o_r, o_bar, total;
  __host__ __device__ FewSmem(int D, int RW, int ng, int nh, int RP, int stages) {
    a_stride = (D + 2 * nh * RP) * 2 + 16;
    kv_stage = 2 * kFewKeys * D * 2;
    r_head = kFewKeys * RP * 2;
    r_stage = ng * r_head;
    const int rings = 4 / RW * stages;
    o_kv = (16 * RW * a_stride + 1023) / 1024 * 1024;
    o_r = o_kv + rings * kv_stage;
    o_bar = o_r + (rings * r_stage + 1023) / 1024 * 1024;
    total = o_bar + 2 * rings * 8 + 16;
  }
};

template <int D, int RW>
__global__ void __launch_bounds__(kFewThreads, 2)
    fna2_paged_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                          const __grid_constant__ CUtensorMap tmRk, const PagedAttnParams p) {
  constexpr int KW = 4 / RW;  // key groups per CTA
  constexpr int DC = D / 64;  // 64-column chunks of a K or V row
  extern __shared__ __align__(1024) uint8_t dsm[];
  if (smem_u32(dsm) & 1023u) {  // the swizzled layouts need it
    if (threadIdx.x == 0) atomicCAS(&g_device_error, 0, kStatusSmemBase);
    return;
  }
  const int split = blockIdx.y;
  const int rb = blockIdx.x % p.row_blocks;
  const int kh = (blockIdx.x / p.row_blocks) % p.kv.hkv;
  const int b = blockIdx.x / (p.row_blocks * p.kv.hkv);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rw = warp % RW, kg = warp / RW;
  const PagedSeq sq = paged_seq(p.bd, b);
  if (!sq.ok && tid == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
  const int rows = sq.n * p.G;                 // row r: head r / n of the group, new token r % n
  const int r0 = rb * 16 * RW;                 // first row of this block
  if (r0 >= rows || rows > p.few_rows) return;
  const int past = sq.len - sq.n;              // may be negative: the first rows then see no key
  // splits of this sequence that hold keys (split 0 always exists: it writes rows that see nothing)
  const int ns = paged_splits(p, sq);
  if (split >= ns) return;
  const int r_last = min(rows, r0 + 16 * RW) - 1;
  // graph heads of the block's rows, local to the group
  const int g_lo = r0 / sq.n, g_hi = min(r_last / sq.n, p.kv.hg - kh * p.G - 1);
  const int ng = max(0, g_hi - g_lo + 1);
  const FewSmem L(D, RW, p.ng_max, p.nh_max, p.RP, p.stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(dsm + L.o_bar) + kg * p.stages;
  uint64_t* empty = full + KW * p.stages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(dsm + L.o_bar + 2 * KW * p.stages * 8);
  if (tid == 0) {
    for (int s = 0; s < KW * p.stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, RW);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  // keys [k_begin, k_end) of this split that some row of the block sees
  int seen = sq.len;
  if (p.causal) {
    // the largest new-token index among the block's rows
    const int i_max = r_last - r0 + 1 >= sq.n || r_last / sq.n != r0 / sq.n ? sq.n - 1 : r_last % sq.n;
    seen = max(0, past + i_max + 1);
  }
  const int k_begin = min(split * p.chunk, seen), k_end = min(seen, k_begin + p.chunk);
  const int n_all = (k_end - k_begin + kFewKeys - 1) / kFewKeys;
  const int n_tiles = n_all > kg ? (n_all - kg + KW - 1) / KW : 0;

  // Ring of the key group: lane l issues box l of a tile (K chunks, V chunks, R_k heads).
  uint8_t* kv_ring = dsm + L.o_kv + kg * p.stages * L.kv_stage;
  uint8_t* r_ring = dsm + L.o_r + kg * p.stages * L.r_stage;
  const int* table = p.kv.table + b * p.kv.table_sb;
  const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
  const bool box = lane < 2 * DC + ng;
  const CUtensorMap* map = lane < DC ? &tmK : lane < 2 * DC ? &tmV : &tmRk;
  const int box_col = lane < 2 * DC ? lane % DC * 64 : 0;
  const int box_head = lane < 2 * DC ? kh : kh * p.G + g_lo + lane - 2 * DC;
  uint8_t* box_dst = lane < 2 * DC ? kv_ring + lane * (kFewKeys * 128) : r_ring + (lane - 2 * DC) * L.r_head;
  const int box_step = lane < 2 * DC ? L.kv_stage : L.r_stage;
  const int tile_bytes = L.kv_stage + ng * L.r_head;
  int issued = 0, i_stage = 0, i_phase = 1;  // empty barriers: the first round passes
  int j_next = k_begin + kg * kFewKeys;
  int page_next = n_tiles > 0 ? __ldg(table + (j_next >> lg)) : 0;
  auto issue = [&]() {
    if (issued >= n_tiles) return;
    const int page = page_next, slot = j_next & mask;
    j_next += KW * kFewKeys;
    ++issued;
    if (issued < n_tiles) page_next = __ldg(table + (j_next >> lg));
    if (RW > 1) mbar_wait(empty + i_stage, i_phase, abort_flag, 131);
    if (lane == 0) mbar_expect_tx(full + i_stage, tile_bytes);
    __syncwarp();
    if (box) tma_load_4d(box_dst + i_stage * box_step, map, full + i_stage, box_col, slot, box_head, page);
    if (++i_stage == p.stages) i_stage = 0, i_phase ^= 1;
  };
  if (rw == 0)
    for (int s = 0; s < p.stages - 1; ++s) issue();

  // A = [q | R~_q hi, lo of the warp's heads] of this warp's 16 rows (rows past the end are zero)
  const int wr0 = r0 + rw * 16;
  const int wg_lo = wr0 / sq.n, wg_hi = min(min(rows - 1, wr0 + 15) / sq.n, p.kv.hg - kh * p.G - 1);
  const int wn = wr0 < rows ? max(0, wg_hi - wg_lo + 1) : 0;
  uint8_t* sa = dsm + rw * 16 * L.a_stride;
  if (kg == 0) {
    for (int e = lane; e < 16 * (D / 8); e += 32) {
      const int row = e / (D / 8), c = e % (D / 8) * 8, r = wr0 + row;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows)
        v = *reinterpret_cast<const uint4*>(p.q + (sq.q0 + r % sq.n) * p.q_st + (kh * p.G + r / sq.n) * p.q_sh + c);
      *reinterpret_cast<uint4*>(sa + row * L.a_stride + c * 2) = v;
    }
    const int rp8 = p.RP / 8;
    for (int e = lane; e < 16 * wn * rp8; e += 32) {
      const int row = e / (wn * rp8), g = e / rp8 % wn, c = e % rp8 * 8, r = wr0 + row;
      uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
      if (r < rows && r / sq.n == wg_lo + g && c < p.kv.rank) {  // block-diagonal: a row holds its own head's R~_q
        const int h = kh * p.G + wg_lo + g;
        split_bias(*reinterpret_cast<const uint4*>(p.rq + (sq.q0 + r % sq.n) * p.rq_st + h * p.rq_sh + c),
                   __ldg(p.gs + h) / p.scale, hi, lo);
      }
      uint8_t* dst = sa + row * L.a_stride + (D + 2 * g * p.RP + c) * 2;
      *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(dst + p.RP * 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
  __syncthreads();

  const int g = lane >> 2, t = lane & 3;
  const int ra = wr0 + g, rc = ra + 8;  // the two rows of this thread's fragments
  // (rows past the end are zero rows that see every key: they are not written)
  auto row_limit = [&](int r) { return min(k_end, p.causal && r < rows ? max(0, past + r % sq.n + 1) : sq.len); };
  const int lim0 = row_limit(ra), lim1 = row_limit(rc);
  // tiles that end at or before every row's limit need no mask
  const int lim_all = __reduce_min_sync(0xffffffffu, min(lim0, lim1));
  const uint32_t a_addr = smem_u32(sa) + ((lane & 7) + ((lane >> 3) & 1) * 8) * L.a_stride + (lane >> 4) * 16;
  uint32_t aq[D / 16][4];  // q fragments stay in registers
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) ldsm_x4(aq[ks], a_addr + ks * 32);
  // ldmatrix addresses within a swizzled tile; rows differ by lane & 7 (+ 8), so the XOR is a lane constant
  const uint32_t k_row = (lane & 7) + (lane >> 4) * 8, k_sel = ((lane >> 3) & 1) * 16;
  const uint32_t v_row = (lane & 7) + ((lane >> 3) & 1) * 8, v_sel = (lane >> 4) * 16;
  const uint32_t k_off = k_row * 128, v_off = kFewKeys * D * 2 + v_row * 128, sw = (lane & 7) * 16;
  const uint32_t r_off = k_row * p.RP * 2, r_sw = p.RP == 16 ? ((k_row >> 2) & 1) * 16 : ((k_row >> 1) & 3) * 16;
  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  // log2 domain: m the maximum that P is relative to, mt this thread's largest logit so far
  float m0 = -INFINITY, m1 = -INFINITY, mt0 = -INFINITY, mt1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float sl2 = p.scale_log2;
  float* lg0 = nullptr;
  float* lg1 = nullptr;
  if (p.logits) {
    float* base = p.logits + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.bd.max_q * p.G * p.logit_sr;
    if (ra < rows) lg0 = base + ra * p.logit_sr;
    if (rc < rows) lg1 = base + rc * p.logit_sr;
  }

  int stage = 0, phase = 0;
  for (int tt = 0; tt < n_tiles; ++tt) {
    __syncwarp();  // (RW == 1) every lane is done with the stage that this issue refills
    if (rw == 0) issue();
    if (!mbar_wait(full + stage, phase, abort_flag, 132)) break;
    uint8_t* kv = kv_ring + stage * L.kv_stage;
    const uint32_t kv_addr = smem_u32(kv);
    const uint32_t rk_addr = smem_u32(r_ring + stage * L.r_stage) + (wg_lo - g_lo) * L.r_head + r_off;
    const int j0 = k_begin + (kg + tt * KW) * kFewKeys;
    if (j0 + kFewKeys > sq.len) {
      // past the sequence's end a page holds anything: V rows become zero (P is 0 there, but 0 * NaN
      // is not); K rows only reach logits that are masked.  The RW warps write the same zeros.
      for (int e = lane; e < (j0 + kFewKeys - sq.len) * 8 * DC; e += 32)
        *reinterpret_cast<uint4*>(kv + kFewKeys * D * 2 + e % DC * (kFewKeys * 128) +
                                  (sq.len - j0) * 128 + e / DC * 16) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t kb[4];
      ldsm_x4(kb, kv_addr + (ks >> 2) * (kFewKeys * 128) + k_off + ((k_sel + (ks & 3) * 32) ^ sw));
      mma_bf16(s0, aq[ks], kb[0], kb[1]);
      mma_bf16(s1, aq[ks], kb[2], kb[3]);
    }
    for (int c = 0; c < wn; ++c)
      for (int ks = 0; ks < p.RP / 16; ++ks) {
        uint32_t a[4], kb[4];
        ldsm_x4(kb, rk_addr + c * L.r_head + ((k_sel + ks * 32) ^ r_sw));
        const uint32_t aw = a_addr + (D + 2 * c * p.RP) * 2 + ks * 32;
        ldsm_x4(a, aw);
        mma_bf16(s0, a, kb[0], kb[1]);
        mma_bf16(s1, a, kb[2], kb[3]);
        ldsm_x4(a, aw + p.RP * 2);
        mma_bf16(s0, a, kb[0], kb[1]);
        mma_bf16(s1, a, kb[2], kb[3]);
      }
    // online softmax: row ra holds x[0..3], row rc x[4..7]; keys j0 + {2t, 2t+1, 8+2t, 9+2t}
    float x[8] = {s0[0], s0[1], s1[0], s1[1], s0[2], s0[3], s1[2], s1[3]};
    if (j0 + kFewKeys > lim_all) {
      const int kk[4] = {j0 + 2 * t, j0 + 2 * t + 1, j0 + 8 + 2 * t, j0 + 9 + 2 * t};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = kk[i] < lim0 ? x[i] : -INFINITY;
        x[4 + i] = kk[i] < lim1 ? x[4 + i] : -INFINITY;
      }
    }
    if (lg0) {
      *reinterpret_cast<float2*>(lg0 + j0 + 2 * t) = make_float2(x[0] * sl2, x[1] * sl2);
      *reinterpret_cast<float2*>(lg0 + j0 + 8 + 2 * t) = make_float2(x[2] * sl2, x[3] * sl2);
    }
    if (lg1) {
      *reinterpret_cast<float2*>(lg1 + j0 + 2 * t) = make_float2(x[4] * sl2, x[5] * sl2);
      *reinterpret_cast<float2*>(lg1 + j0 + 8 + 2 * t) = make_float2(x[6] * sl2, x[7] * sl2);
    }
    float mx0 = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * sl2;
    float mx1 = fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])) * sl2;
    mt0 = fmaxf(mt0, mx0), mt1 = fmaxf(mt1, mx1);
    // the maximum in use moves only when some logit is above it by more than 2^8 (P stays in range)
    if (__any_sync(0xffffffffu, mx0 > m0 + 8.f || mx1 > m1 + 8.f)) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
      const float c0 = n0 == -INFINITY ? 1.f : ex2(m0 - n0), c1 = n1 == -INFINITY ? 1.f : ex2(m1 - n1);
      m0 = n0, m1 = n1;
      l0 *= c0, l1 *= c1;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) acc[i][0] *= c0, acc[i][1] *= c0, acc[i][2] *= c1, acc[i][3] *= c1;
    }
    const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ex2(fmaf(x[i], sl2, -b0)), x[4 + i] = ex2(fmaf(x[4 + i], sl2, -b1));
    l0 += (x[0] + x[1]) + (x[2] + x[3]);
    l1 += (x[4] + x[5]) + (x[6] + x[7]);
    const uint32_t pa[4] = {pack_bf16(x[0], x[1]), pack_bf16(x[4], x[5]), pack_bf16(x[2], x[3]),
                            pack_bf16(x[6], x[7])};
#pragma unroll
    for (int d16 = 0; d16 < D / 16; ++d16) {
      uint32_t vb[4];
      ldsm_x4_t(vb, kv_addr + (d16 >> 2) * (kFewKeys * 128) + v_off + ((v_sel + (d16 & 3) * 32) ^ sw));
      mma_bf16(acc[2 * d16], pa, vb[0], vb[1]);
      mma_bf16(acc[2 * d16 + 1], pa, vb[2], vb[3]);
    }
    if (RW > 1) {
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + stage);
    }
    if (++stage == p.stages) stage = 0, phase ^= 1;
  }
  // sums and the true maximum over the row's four lanes; everything relative to that maximum
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    mt0 = fmaxf(mt0, __shfl_xor_sync(0xffffffffu, mt0, o));
    mt1 = fmaxf(mt1, __shfl_xor_sync(0xffffffffu, mt1, o));
  }
  const float f0 = mt0 == -INFINITY ? 0.f : ex2(m0 - mt0), f1 = mt1 == -INFINITY ? 0.f : ex2(m1 - mt1);

  // join the KW key groups through shared memory (all rings are idle)
  __syncthreads();
  float* cm = reinterpret_cast<float*>(dsm);  // [KW][16 RW] m
  float* cl = cm + 64;                        // [KW][16 RW] l
  float* co = cl + 64;                        // [KW][16 RW][D] acc
  const int slot = kg * 16 * RW + rw * 16 + g;
  if (t == 0) {
    cm[slot] = mt0, cm[slot + 8] = mt1;
    cl[slot] = l0 * f0, cl[slot + 8] = l1 * f1;
  }
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    *reinterpret_cast<float2*>(co + slot * D + i * 8 + 2 * t) = make_float2(acc[i][0] * f0, acc[i][1] * f0);
    *reinterpret_cast<float2*>(co + (slot + 8) * D + i * 8 + 2 * t) = make_float2(acc[i][2] * f1, acc[i][3] * f1);
  }
  __syncthreads();
  const int nr = r_last - r0 + 1;
  for (int e = tid; e < nr * (D / 4); e += kFewThreads) {
    const int row = e / (D / 4), d = e % (D / 4) * 4, r = r0 + row;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < KW; ++w) M = fmaxf(M, cm[w * 16 * RW + row]);
    float Ls = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float f = ex2(cm[w * 16 * RW + row] - M);
        const float4 a = *reinterpret_cast<const float4*>(co + (w * 16 * RW + row) * D + d);
        Ls += cl[w * 16 * RW + row] * f;
        O.x += a.x * f, O.y += a.y * f, O.z += a.z * f, O.w += a.w * f;
      }
    }
    const int64_t tok = sq.q0 + r % sq.n;
    const int h = kh * p.G + r / sq.n;
    const int64_t w = (tok * p.H + h) * p.ns + split;
    if (d == 0 && p.ws_ml) p.ws_ml[w] = make_float2(M, Ls);
    if (ns == 1) {
      const float inv = 1.f / (Ls + kEps);
      *reinterpret_cast<uint2*>(p.out + tok * p.o_st + h * p.o_sh + d) =
          make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
      if (d == 0 && p.lse) p.lse[h * p.lse_sh + tok] = M == -INFINITY ? M : (M + log2f(Ls + kEps)) * kLn2;
    } else {
      *reinterpret_cast<float4*>(p.ws_acc + w * D + d) = O;
    }
  }
}

// Joins the splits of one (token, query head), a warp each: rescale to the
// common max, O = acc / (l + 1e-6), LSE = m + log(l + 1e-6).
template <int D>
__global__ void __launch_bounds__(128) fna2_paged_join_kernel(const PagedAttnParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t th = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int64_t tok = th / p.H;
  const int h = static_cast<int>(th % p.H);
  if (tok >= p.bd.T) return;
  const int b = warp_seq_of(p.bd.cu, p.bd.B, tok, lane);
  if (b < 0) return;
  const PagedSeq sq = paged_seq(p.bd, b);
  const int ns = paged_splits(p, sq);
  if (!sq.ok || ns <= 1) return;  // written by the attention kernel
  const float2* ml = p.ws_ml + th * p.ns;
  float M = -INFINITY;
  for (int s = 0; s < ns; ++s) M = fmaxf(M, ml[s].x);
  float Ls = 0.f;
  float O[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) O[i] = 0.f;
  if (M != -INFINITY)
    for (int s = 0; s < ns; ++s) {
      const float2 v = ml[s];
      if (v.x == -INFINITY) continue;
      const float f = exp2f(v.x - M);
      Ls += v.y * f;
      const float* a = p.ws_acc + (th * p.ns + s) * D + lane * (D / 32);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) O[i] += a[i] * f;
    }
  const float inv = 1.f / (Ls + kEps);
  __nv_bfloat16* o = p.out + tok * p.o_st + h * p.o_sh + lane * (D / 32);
#pragma unroll
  for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<uint32_t*>(o + i) = pack_bf16(O[i] * inv, O[i + 1] * inv);
  if (lane == 0 && p.lse) p.lse[h * p.lse_sh + tok] = M == -INFINITY ? M : (M + log2f(Ls + kEps)) * kLn2;
}

// Key weights of a call whose logits were kept: w[b, kh, j] += sum over the rows
// of 2^(x - LSE).  One thread per key.
constexpr int kLogitThreads = 256;
__global__ void __launch_bounds__(kLogitThreads) fna2_paged_logit_weights_kernel(const PagedAttnParams p) {
  const int kh = blockIdx.y, b = blockIdx.z;
  const PagedSeq sq = paged_seq(p.bd, b);
  if (static_cast<int>(blockIdx.x) * kLogitThreads >= sq.len) return;
  const int j = blockIdx.x * kLogitThreads + threadIdx.x, rows = sq.n * p.G;
  const int ns = paged_splits(p, sq), past = sq.len - sq.n;
  __shared__ float s_lse[kLogitThreads];
  float w = 0.f;
  const float* x = p.logits + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.bd.max_q * p.G * p.logit_sr + j;
  for (int base = 0; base < rows; base += kLogitThreads) {
    __syncthreads();
    if (base + static_cast<int>(threadIdx.x) < rows) {
      const int r = base + threadIdx.x;
      const int64_t th = static_cast<int64_t>(sq.q0 + r % sq.n) * p.H + kh * p.G + r / sq.n;
      float M = -INFINITY, Ls = 0.f;
      for (int s = 0; s < ns; ++s) M = fmaxf(M, p.ws_ml[th * p.ns + s].x);
      if (M != -INFINITY)
        for (int s = 0; s < ns; ++s) Ls += p.ws_ml[th * p.ns + s].y * exp2f(p.ws_ml[th * p.ns + s].x - M);
      s_lse[threadIdx.x] = M == -INFINITY ? INFINITY : M + log2f(Ls + kEps);  // a row without weight adds 0
    }
    __syncthreads();
    if (j < sq.len) {
      const int n = min(kLogitThreads, rows - base);
      for (int r = 0; r < n; ++r)
        if (!p.causal || j <= past + (base + r) % sq.n) w += exp2f(x[(base + r) * p.logit_sr] - s_lse[r]);
    }
  }
  if (j < sq.len) p.kw[b * p.kw_sb + kh * p.kw_sh + j] += w;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct FewMaps {
  CUtensorMap k, v, rk;
};

template <int D, int RW>
cudaError_t launch_paged_few_t(const FewMaps& m, const PagedAttnParams& p, size_t smem, cudaStream_t stream) {
  auto kern = fna2_paged_few_kernel<D, RW>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  const dim3 grid(p.bd.B * p.kv.hkv * p.row_blocks, (std::max(1, p.bd.max_k) + p.chunk - 1) / p.chunk);
  kern<<<grid, kFewThreads, smem, stream>>>(m.k, m.v, m.rk, p);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_paged_few_d(const FewMaps& m, const PagedAttnParams& p, int RW, size_t smem, cudaStream_t stream) {
  return RW == 1   ? launch_paged_few_t<D, 1>(m, p, smem, stream)
         : RW == 2 ? launch_paged_few_t<D, 2>(m, p, smem, stream)
                   : launch_paged_few_t<D, 4>(m, p, smem, stream);
}

inline cudaError_t launch_paged_few(const FewMaps& m, const PagedAttnParams& p, int D, int RW, size_t smem,
                                    cudaStream_t stream) {
  return D == 128 ? launch_paged_few_d<128>(m, p, RW, smem, stream) : launch_paged_few_d<64>(m, p, RW, smem, stream);
}

// What follows the attention kernels: the join of the splits and the weights from kept logits.
inline cudaError_t launch_paged_tail(const PagedAttnParams& p, int D, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (p.ns > 1) {
    const int64_t blocks = (static_cast<int64_t>(p.bd.T) * p.H + 3) / 4;
    if (D == 128)
      fna2_paged_join_kernel<128><<<static_cast<unsigned>(blocks), 128, 0, stream>>>(p);
    else
      fna2_paged_join_kernel<64><<<static_cast<unsigned>(blocks), 128, 0, stream>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (p.logits) {
    const dim3 grid((p.bd.max_k + kLogitThreads - 1) / kLogitThreads, p.kv.hkv, p.bd.B);
    fna2_paged_logit_weights_kernel<<<grid, kLogitThreads, 0, stream>>>(p);
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace fna2
