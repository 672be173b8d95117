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
// bf16 for P V, as in the prefill kernels; the row sums use the unrounded P.  The
// bf16 output then lies 2.3e-3 (2-norm) from the 64-bit one, of which 1.7e-3 is its own
// rounding; the rest of P as a second bf16 operand would leave only that, for 2 to 7 %
// of the time (131,071 keys: 332 -> 354 us).
//
// A unit is 64/RW keys of a sequence.  The units of all sequences, in order, are
// cut into equal runs, whatever the lengths, and each run is taken by one CTA for
// every (KV head, block of 16 RW query rows): as many runs as fill the GPU once, and
// all heads' rows of the same keys are read at the same time (in a pool laid out by
// token they are neighbours in memory; with runs cut per head instead, DRAM gave
// 5.8 instead of 6.8 TB/s).  A run covers the end of one sequence, whole ones and the
// start of another, and fna2_paged_few_join_kernel joins the sequences that were
// cut.  A query row is (query head of the KV group, new token), head-major,
// so that the 16 rows of a warp span few heads.  4 warps: RW row blocks x 4/RW key
// groups; a key group streams its own 16-key tiles through a ring in shared memory
// that its RW warps fill with asynchronous copies (16 bytes a lane, whole rows an
// instruction, rows swizzled for conflict-free ldmatrix) and read together
// (mma.sync m16n8k16, fp32 accumulation, online softmax in registers).  16 keys never
// cross a page, so a tile needs one page lookup and a lane's addresses are one base
// and constant steps.  (One TMA box per 64 columns and head instead: each costs the
// issuing warp about 110 clk, 580 of the 1800 clk of a tile; a general address per
// copy: 820 instructions a tile.)
// Bound: HBM; each cached key is read once per row block.  One token of one sequence of
// 131,071 keys, 32 separate heads, D = 128, rank 16: 332 us with the join, 6.9 TB/s; of 64
// sequences of up to 4,096 keys, 8 KV heads of 4: 117 us, 5.8 TB/s, the join and the key
// weights 16 more.  Short sequences are bound by latency (the scan, a page lookup, the first
// tiles) and by the join's second grid (16 sequences of up to 2,048 keys, 4 KV heads: 27 us,
// of which HBM 7).
#include "fna2_paged.cuh"

namespace fna2 {

struct PagedAttnParams {
  PagedPool kv;
  PagedBounds bd;
  int H, G;       // query heads, query heads per KV head
  int RP;         // rank rounded up to 16 or 32
  int causal;
  float scale, scale_log2, inv_scale;
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const __nv_bfloat16* rq;
  int64_t rq_st, rq_sh;
  const float* gs;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  float* lse;  // [H][lse_sh], or NULL
  int64_t lse_sh;
  // tensor-core kernel: its splits of a sequence, at most ns of them
  int ns;
  float* ws_acc;      // [(t * H + h) * ns + split][D]: unnormalised output of a split
  float2* ws_ml;      // [(t * H + h) * ns + split]: its row max (log2 domain) and sum
  // mma.sync kernel: a CTA's first and last sequence may be parts of one
  float* part_acc;    // [(cta * 2 + first or last) * block_rows + row][D]
  float2* part_ml;    // [(cta * 2 + first or last) * block_rows + row]
  int64_t* prefix;    // [B + 1] units before each sequence, then their number
  float* lse2;        // [t * H + h] log2-domain LSE of the rows of sequences not cut (kept with logits)
  float* logits;      // key weights: [((b * HKV + kh) * max_q * G + row)][logit_sr] log2-domain logits, or NULL
  int64_t logit_sr;
  float* kw;          // key weights, added to: [b * kw_sb + kh * kw_sh + j]
  int64_t kw_sb, kw_sh;
  int block_rows;     // 16 RW
  int unit_keys;      // 64 / RW
  int whole;          // sequences are not cut (they are short): a unit is a sequence
  int runs;           // at most
  int row_blocks;     // row blocks per KV head; CTA = (run * HKV + KV head) * row_blocks + row block
  int ng_max, stages;
  // Sequences of more than few_rows query rows (new tokens x query heads of a KV head) go to
  // fna2_paged_many_kernel, the others to fna2_paged_few_kernel; a call launches those it may need.
  int few_rows;
  int chunk_many, many_items;  // keys per split there, upper bound on its (query tile pair, split) items
  int after_many;  // the few-row kernel runs after the tensor-core kernel, on the SMs that it leaves
};

// Units of one sequence in the mma.sync kernel: 0 when it is not this kernel's.
__device__ __forceinline__ int few_units(const PagedAttnParams& p, const PagedSeq& s) {
  const int rows = s.n * p.G;
  if (rows == 0 || rows > p.few_rows) return 0;
  return p.whole ? 1 : max(1, (s.len + p.unit_keys - 1) / p.unit_keys);
}
// Runs that share U units (each takes at least one); the first unit of run c; the run of unit u.
__device__ __forceinline__ int few_runs(const PagedAttnParams& p, int64_t U) {
  return static_cast<int>(min(static_cast<int64_t>(p.runs), max(U, static_cast<int64_t>(1))));
}
__device__ __forceinline__ int64_t few_first(int64_t U, int C, int c) { return U * c / C; }
__device__ __forceinline__ int few_run_of(int64_t U, int C, int64_t u) { return static_cast<int>(((u + 1) * C - 1) / U); }

// New tokens, and query rows per KV head (new tokens x query heads of the group), up to which a sequence is
// streamed by the mma.sync kernel.  Its time goes by KV heads and blocks of up to 64 rows; the tensor-core
// kernel's by query heads and 128-row tiles, however few rows fill them.  8 sequences of 100 to 4,000 keys, 16
// query heads with bias of rank 16, D = 128, mma.sync against tensor-core kernel: 32 tokens of 4 KV heads (128
// rows) 54 / 71 us, 48 tokens 70 / 64; of 16 KV heads, 32 tokens (32 rows) 53 / 74, 48 tokens 83 / 65.  With 2
// KV heads the limit is low: 16 tokens (128 rows) 35 / 68, 24 tokens 47 / 70, 32 tokens 54 / 71.
constexpr int kFewTokens = 32;
constexpr int kFewRows = 128;
// Rows up to which the mma.sync kernel keeps its logits for the key weights, rather than have them formed
// again by the key weights' kernels: 16 sequences of 1,000 to 4,000 keys, 8 KV heads, D = 128, kept / formed
// again: 4 rows 53 / 82 us, 16 rows 75 / 97 us, 32 rows 88 / 99 us, 64 rows 138 / 129 us.
constexpr int kLogitRows = 32;
// ... rows in a call that has longer sequences: its few-row ones mostly add one token, in one 16-row block
// (26 sequences, chunks of up to 500 tokens next to single ones: 123 us; up to 32 rows 158, 64 rows 250.  Measured
// with one query head per KV head; groups of more than 16 leave the kernel nothing in such a call).
constexpr int kFewRowsMixed = 16;
// Dynamic shared memory of which two CTAs fit on an SM (228 KB, 1 KB reserved per CTA).
constexpr int kHalfSmem = 113 * 1024;

constexpr int kFewThreads = 128;
constexpr int kFewKeys = 16;  // keys per tile

// Shared-memory geometry (host and device agree on it): [A of the RW row blocks | K and V ring of
// the key groups | R_k ring | m, l and accumulators of the key groups | scan]; ng: graph heads
// of a block's rows.
struct FewSmem {
  int a_stride, kv_stage, r_head, r_stage, o_kv, o_r, o_join, o_bar, total;
  // (of the row blocks' rows only `rows`, their bound, have a place in A and are joined)
  __host__ __device__ FewSmem(int D, int RW, int ng, int RP, int stages, int rows) {
    a_stride = (D + 2 * RP) * 2 + 16;
    kv_stage = 2 * kFewKeys * D * 2;
    r_head = kFewKeys * RP * 2;
    r_stage = ng * r_head;
    const int rings = 4 / RW * stages;
    const int blocks = rows < 16 * RW ? (rows + 15) / 16 : RW;  // row blocks that can hold a row
    o_kv = (16 * blocks * a_stride + 1023) / 1024 * 1024;
    o_r = o_kv + rings * kv_stage;
    o_join = o_r + (rings * r_stage + 1023) / 1024 * 1024;
    o_bar = o_join + 512 + 4 / RW * (rows < 16 * RW ? rows : 16 * RW) * D * 4;
    total = o_bar + 80;
  }
};

// Rendezvous of the RW warps of a key group (named barrier 1 + group).
template <int RW>
__device__ __forceinline__ void group_sync(int kg) {
  if (RW == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * RW) : "memory");
}

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void few_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void few_cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// d = a b + c
__device__ __forceinline__ void mma_bf16_from(float (&d)[4], const float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Factor of a part with maximum m in a row of maximum M (log2 domain).  A part that saw no key has m = -inf and
// sum 0; one whose logits are all NaN has m = -inf and sum NaN, which stays.
__device__ __forceinline__ float part_factor(float m, float M) { return m == M ? 1.f : ex2(m - M); }

// Four columns of a finished row: O = acc / (l + 1e-6), LSE = m + log(l + 1e-6): 0 and -inf where no key was seen.
template <int D>
__device__ __forceinline__ void few_store(const PagedAttnParams& p, int64_t tok, int h, int d, float M, float Ls,
                                          const float4& O) {
  const float inv = 1.f / (Ls + kEps);
  *reinterpret_cast<uint2*>(p.out + tok * p.o_st + h * p.o_sh + d) =
      make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
  if (d == 0) {
    const float lse2 = M + log2f(Ls + kEps);
    if (p.lse) p.lse[h * p.lse_sh + tok] = lse2 * kLn2;
    if (p.lse2) p.lse2[tok * p.H + h] = lse2;
  }
}

template <int D, int RW>
__global__ void __launch_bounds__(kFewThreads, 2) fna2_paged_few_kernel(const PagedAttnParams p) {
  constexpr int KW = 4 / RW;  // key groups per CTA
  if (!p.after_many) pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t dsm[];
  const int cta = blockIdx.x, lanes = p.kv.hkv * p.row_blocks, run = cta / lanes;
  const int kh = cta % lanes / p.row_blocks, r0 = cta % p.row_blocks * (16 * RW);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rw = warp % RW, kg = warp / RW;
  const FewSmem L(D, RW, p.ng_max, p.RP, p.stages, p.few_rows);
  int64_t* s_scan = reinterpret_cast<int64_t*>(dsm + L.o_bar);  // [4] warps' sums, [4]: units before the first sequence
  int* s_first = reinterpret_cast<int*>(s_scan + 5);            // first sequence: b, q0, n, len

  // R_k ring: columns [rank, RP) of every head are zero, and stay so.
  uint8_t* r_ring = dsm + L.o_r + kg * p.stages * L.r_stage;
  const int rp8 = p.RP / 8, r8 = p.kv.rank / 8;
  if (r8 != rp8) {
    const int n = 4 / RW * p.stages * p.ng_max * 16;  // rows of all rings
    for (int e = tid; e < n * (rp8 - r8); e += kFewThreads) {
      const int row = e % n, c = r8 + e / n, sw = p.RP == 16 ? (row >> 2) & 1 : (row >> 1) & 3;
      *reinterpret_cast<uint4*>(dsm + L.o_r + row * p.RP * 2 + (c ^ sw) * 16) = make_uint4(0, 0, 0, 0);
    }
  }

  // Number of units U, this CTA's run [u_beg, u_end) of them, and the sequence that its first unit is in:
  // a scan over the sequences, 128 a round (a second pass over the later rounds when there are more).
  int64_t U = 0, pre0 = 0;
  int units0 = 0;
  PagedSeq sq0{0, 0, 0, false};
  auto scan = [&](int base, PagedSeq* s, int* units) {
    const int b = base + tid;
    *units = 0;
    if (b < p.bd.B) {
      *s = paged_seq(p.bd, b);
      if (!s->ok && cta == 0) atomicCAS(&g_device_error, 0, kStatusBadSeqPaged);
      *units = few_units(p, *s);
    }
    int64_t incl = *units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int64_t pre = U + incl - *units;
    for (int w = 0; w < warp; ++w) pre += s_scan[w];
    U += s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3];
    __syncthreads();
    if (cta == 0 && b < p.bd.B && p.prefix) p.prefix[b] = pre;
    return pre;
  };
  pre0 = scan(0, &sq0, &units0);
  const int64_t U0 = U;
  for (int base = kFewThreads; base < p.bd.B; base += kFewThreads) {
    PagedSeq s;
    int units;
    scan(base, &s, &units);
  }
  const int C = few_runs(p, U);
  const int64_t U_all = U, u_beg = few_first(U, C, min(run, C)), u_end = few_first(U, C, min(run + 1, C));
  if (cta == 0 && tid == 0 && p.prefix) p.prefix[p.bd.B] = U;
  if (u_beg == u_end) {
    pdl_wait();
    return;
  }
  auto found = [&](int b, const PagedSeq& s, int units, int64_t pre) {
    if (units > 0 && pre <= u_beg && u_beg < pre + units)
      s_first[0] = b, s_first[1] = s.q0, s_first[2] = s.n, s_first[3] = s.len, s_scan[4] = pre;
  };
  found(tid, sq0, units0, pre0);
  U = U0;
  for (int base = kFewThreads; base < p.bd.B && U <= u_beg && U < U_all; base += kFewThreads) {
    PagedSeq s;
    int units;
    const int64_t pre = scan(base, &s, &units);
    found(base + tid, s, units, pre);
  }
  __syncthreads();

  // Current sequence: units [o_beg, o_end) of it.
  int64_t u = u_beg, pre = s_scan[4];
  int b = s_first[0];
  PagedSeq sq{s_first[1], s_first[2], s_first[3], true};
  int units = few_units(p, sq), rows, r_last, o_beg, o_end, past, g_lo, ng, k_begin, k_end, n_tiles;
  const int* table;
  auto segment = [&]() {
    o_beg = static_cast<int>(u - pre);
    o_end = static_cast<int>(min(static_cast<int64_t>(units), o_beg + (u_end - u)));
    rows = sq.n * p.G;                          // row r: head r / n of the group, new token r % n
    r_last = min(rows, r0 + 16 * RW) - 1;       // below r0: this block has no row of the sequence
    past = sq.len - sq.n;                       // may be negative: the first rows then see no key
    // graph heads of the block's rows, local to the group
    g_lo = r0 / sq.n;
    ng = max(0, min(r_last / sq.n, p.kv.hg - kh * p.G - 1) - g_lo + 1);
    // keys that some row of the block sees
    int seen = sq.len;
    if (p.causal) {
      const int i_max = r_last - r0 + 1 >= sq.n || r_last / sq.n != r0 / sq.n ? sq.n - 1 : r_last % sq.n;
      seen = max(0, past + i_max + 1);
    }
    if (r0 >= rows) seen = 0;
    k_begin = p.whole ? 0 : min(o_beg * p.unit_keys, seen);
    k_end = p.whole ? seen : min(o_end * p.unit_keys, seen);
    const int n_all = (k_end - k_begin + kFewKeys - 1) / kFewKeys;
    n_tiles = n_all > kg ? (n_all - kg + KW - 1) / KW : 0;
    table = p.kv.table + b * p.kv.table_sb;
  };
  segment();

  // Ring of the key group.  K and V: lane l copies 16-byte piece l % PPR of row row0 + k RW RPI, in turn
  // k; piece c of row r lies at chunk c ^ (r & 7) of its 128 bytes.  R_k: piece x of row lane % 16.
  constexpr int PPR = D / 8, RPI = 32 / PPR, NI = 16 / (RW * RPI), STEP = RW * RPI;
  uint8_t* kv_ring = dsm + L.o_kv + kg * p.stages * L.kv_stage;
  const int lg = p.kv.page_log2, mask = (1 << lg) - 1;
  const int row0 = rw * RPI + lane / PPR, pc = lane % PPR, r_row = lane % 16, r_lg = p.RP == 16 ? 1 : 2;
  const uint32_t d_lane = (pc >> 3) * (kFewKeys * 128) + row0 * 128 + ((pc ^ row0) & 7) * 16;
  const uint32_t dr_lane = r_row * p.RP * 2;
  const int dr_sw = p.RP == 16 ? (r_row >> 2) & 1 : (r_row >> 1) & 3;
  const __nv_bfloat16* k_lane = p.kv.k.ptr + kh * p.kv.k.sh + row0 * p.kv.k.st + pc * 8;
  const __nv_bfloat16* v_lane = p.kv.v.ptr + kh * p.kv.v.sh + row0 * p.kv.v.st + pc * 8;
  int issued = 0, i_stage = 0, j_next = 0, page_next = 0;
  auto issue = [&]() {
    if (issued < n_tiles) {
      const int page = page_next, slot = j_next & mask, j0 = j_next;
      j_next += KW * kFewKeys;
      if (++issued < n_tiles) page_next = __ldg(table + (j_next >> lg));
      const uint32_t dk = smem_u32(kv_ring + i_stage * L.kv_stage) + d_lane;
      const uint32_t dr = smem_u32(r_ring + i_stage * L.r_stage) + dr_lane;
      // rows past the sequence's end are zero-filled: what a page holds there is never used
      const int nv = page >= 0 && page < p.kv.pages ? min(kFewKeys, sq.len - j0) : 0;
      const int64_t pg = nv > 0 ? page : 0;
      const __nv_bfloat16* ks = k_lane + pg * p.kv.k.sp + slot * p.kv.k.st;
      const __nv_bfloat16* vs = v_lane + pg * p.kv.v.sp + slot * p.kv.v.st;
      if (nv == kFewKeys) {
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          const uint32_t d = (dk ^ ((k * STEP & 7) * 16)) + k * STEP * 128;
          few_cp16(d, ks);
          few_cp16(d + kFewKeys * D * 2, vs);
          ks += STEP * p.kv.k.st, vs += STEP * p.kv.v.st;
        }
      } else {
        if (nv == 0 && lane == 0) check_page(p.kv, page);
        for (int k = 0; k < NI; ++k) {
          const uint32_t d = (dk ^ ((k * STEP & 7) * 16)) + k * STEP * 128;
          const bool valid = row0 + k * STEP < nv;
          few_cp16(d, valid ? ks : p.kv.k.ptr, valid);
          few_cp16(d + kFewKeys * D * 2, valid ? vs : p.kv.v.ptr, valid);
          ks += STEP * p.kv.k.st, vs += STEP * p.kv.v.st;
        }
      }
      if (ng > 0) {
        const bool valid = r_row < nv;
        const __nv_bfloat16* rs = p.kv.rk.ptr + (kh * p.G + g_lo) * p.kv.rk.sh + pg * p.kv.rk.sp + (slot + r_row) * p.kv.rk.st;
        for (int x = lane / 16 + 2 * rw; x < ng << r_lg; x += 2 * RW) {
          const int hh = x >> r_lg, c = x & (rp8 - 1);
          if (c < r8)
            few_cp16(dr + hh * L.r_head + (c ^ dr_sw) * 16, valid ? rs + hh * p.kv.rk.sh + c * 8 : p.kv.rk.ptr, valid);
        }
      }
      if (++i_stage == p.stages) i_stage = 0;
    }
    dec_commit();
  };
  // The first tiles of a sequence; the ring is empty here.
  auto start = [&]() {
    issued = 0;
    j_next = k_begin + kg * kFewKeys;
    if (n_tiles > 0) page_next = __ldg(table + (j_next >> lg));
    for (int s = 0; s < p.stages - 1; ++s) issue();
  };
  start();

  int stage = 0;
  while (true) {
  // A = [q | R~_q hi, lo] of the row blocks' 16 rows each (rows past the end are zero)
  const int wr0 = r0 + rw * 16;
  const int wg_lo = wr0 / sq.n, wg_hi = min(min(rows - 1, wr0 + 15) / sq.n, p.kv.hg - kh * p.G - 1);
  const int wn = wr0 < rows ? max(0, wg_hi - wg_lo + 1) : 0;
  // (a warp that can hold no row computes on the first one's, for nobody: skipping cost the others 2 %)
  const bool holds = RW == 1 || rw * 16 < p.few_rows;
  uint8_t* sa = dsm + (holds ? rw : 0) * 16 * L.a_stride;
  if (holds) {
    constexpr int TPR = 2 * KW;  // threads per row
    const int part = kg * 32 + lane, row = part / TPR, sub = part % TPR, r = wr0 + row;
    const bool real = r < rows;
    const int hh = real ? r / sq.n : 0, h = kh * p.G + hh;
    const int64_t tok = sq.q0 + (r - hh * sq.n);
    uint4 v[D / 8 / TPR];
#pragma unroll
    for (int k = 0; k < D / 8 / TPR; ++k)
      v[k] = real ? *reinterpret_cast<const uint4*>(p.q + tok * p.q_st + h * p.q_sh + (sub + k * TPR) * 8)
                  : make_uint4(0, 0, 0, 0);
    const bool graph = real && h < p.kv.hg;
    const float f = graph ? __ldg(p.gs + h) * p.inv_scale : 0.f;
    if (wn > 0)
      for (int c = sub; c < rp8; c += TPR) {
        uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
        if (graph && c < r8)
          split_bias(*reinterpret_cast<const uint4*>(p.rq + tok * p.rq_st + h * p.rq_sh + c * 8), f, hi, lo);
        uint8_t* dst = sa + row * L.a_stride + (D + c * 8) * 2;
        *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + p.RP * 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
#pragma unroll
    for (int k = 0; k < D / 8 / TPR; ++k) *reinterpret_cast<uint4*>(sa + row * L.a_stride + (sub + k * TPR) * 16) = v[k];
  }
  __syncthreads();

  const int g = lane >> 2, t = lane & 3;
  const int ra = wr0 + g, rc = ra + 8;  // the two rows of this thread's fragments
  const int head_a = ra / sq.n - wg_lo, head_c = rc / sq.n - wg_lo;
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

  for (int tt = 0; tt < n_tiles; ++tt) {
    group_sync<RW>(kg);      // everyone is done with the stage that this issue refills
    issue();
    dec_wait(p.stages - 1);  // this thread's pieces of tile tt have landed
    group_sync<RW>(kg);      // and so have the others'
    const uint32_t kv_addr = smem_u32(kv_ring + stage * L.kv_stage);
    const uint32_t rk_addr = smem_u32(r_ring + stage * L.r_stage) + (wg_lo - g_lo) * L.r_head + r_off;
    const int j0 = k_begin + (kg + tt * KW) * kFewKeys;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t kb[4];
      ldsm_x4(kb, kv_addr + (ks >> 2) * (kFewKeys * 128) + k_off + ((k_sel + (ks & 3) * 32) ^ sw));
      mma_bf16(s0, aq[ks], kb[0], kb[1]);
      mma_bf16(s1, aq[ks], kb[2], kb[3]);
    }
    // The bias: the 16 rows against one head's R_k at a time, of which that head's rows take the sum.  (Zeros
    // in the other heads' columns of one wide A instead would carry an infinity or NaN of one head's R_k into
    // the other heads' rows: 0 * NaN.)
    for (int c = 0; c < wn; ++c) {
      float t0[4], t1[4];
      uint32_t a[4], kb[4];
      ldsm_x4(kb, rk_addr + c * L.r_head + (k_sel ^ r_sw));
      ldsm_x4(a, a_addr + D * 2);
      mma_bf16_from(t0, s0, a, kb[0], kb[1]);
      mma_bf16_from(t1, s1, a, kb[2], kb[3]);
      ldsm_x4(a, a_addr + (D + p.RP) * 2);
      mma_bf16(t0, a, kb[0], kb[1]);
      mma_bf16(t1, a, kb[2], kb[3]);
      if (p.RP == 32) {
        ldsm_x4(kb, rk_addr + c * L.r_head + ((k_sel + 32) ^ r_sw));
        ldsm_x4(a, a_addr + D * 2 + 32);
        mma_bf16(t0, a, kb[0], kb[1]);
        mma_bf16(t1, a, kb[2], kb[3]);
        ldsm_x4(a, a_addr + (D + 32) * 2 + 32);
        mma_bf16(t0, a, kb[0], kb[1]);
        mma_bf16(t1, a, kb[2], kb[3]);
      }
      const bool ma = head_a == c, mc = head_c == c;
      s0[0] = ma ? t0[0] : s0[0], s0[1] = ma ? t0[1] : s0[1], s1[0] = ma ? t1[0] : s1[0], s1[1] = ma ? t1[1] : s1[1];
      s0[2] = mc ? t0[2] : s0[2], s0[3] = mc ? t0[3] : s0[3], s1[2] = mc ? t1[2] : s1[2], s1[3] = mc ? t1[3] : s1[3];
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
    if (++stage == p.stages) stage = 0;
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

  // join the KW key groups through shared memory
  float* cm = reinterpret_cast<float*>(dsm + L.o_join);  // [KW][16 RW] m
  float* cl = cm + 64;                                   // [KW][16 RW] l
  float* co = cl + 64;                                   // [KW][rows kept][D] acc
  const int kept = min(16 * RW, p.few_rows), la = rw * 16 + g;
  if (t == 0) {
    cm[kg * 16 * RW + la] = mt0, cm[kg * 16 * RW + la + 8] = mt1;
    cl[kg * 16 * RW + la] = l0 * f0, cl[kg * 16 * RW + la + 8] = l1 * f1;
  }
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    if (la < kept)
      *reinterpret_cast<float2*>(co + (kg * kept + la) * D + i * 8 + 2 * t) = make_float2(acc[i][0] * f0, acc[i][1] * f0);
    if (la + 8 < kept)
      *reinterpret_cast<float2*>(co + (kg * kept + la + 8) * D + i * 8 + 2 * t) =
          make_float2(acc[i][2] * f1, acc[i][3] * f1);
  }
  // the next sequence's loads start before this one's results are written
  const bool cut = o_end - o_beg != units;
  const int nr = r_last - r0 + 1, part = (cta * 2 + (u == u_beg ? 0 : 1)) * (16 * RW);
  const int out_n = sq.n;
  const int64_t out_q0 = sq.q0;
  u += o_end - o_beg;
  const bool more = u < u_end;
  if (more) {
    while (u - pre >= units) {
      pre += units;
      sq = paged_seq(p.bd, ++b);
      units = few_units(p, sq);
    }
    segment();
    group_sync<RW>(kg);  // everyone is done with the ring
    start();
  }
  __syncthreads();
  for (int e = tid; e < nr * (D / 4); e += kFewThreads) {
    const int row = e / (D / 4), d = e % (D / 4) * 4, r = r0 + row;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < KW; ++w) M = fmaxf(M, cm[w * 16 * RW + row]);
    float Ls = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float f = part_factor(cm[w * 16 * RW + row], M);
      const float4 a = *reinterpret_cast<const float4*>(co + (w * kept + row) * D + d);
      Ls += cl[w * 16 * RW + row] * f;
      O.x += a.x * f, O.y += a.y * f, O.z += a.z * f, O.w += a.w * f;
    }
    if (cut) {
      *reinterpret_cast<float4*>(p.part_acc + static_cast<int64_t>(part + row) * D + d) = O;
      if (d == 0) p.part_ml[part + row] = make_float2(M, Ls);
    } else {
      few_store<D>(p, out_q0 + r % out_n, kh * p.G + r / out_n, d, M, Ls, O);
    }
  }
  if (!more) break;
  }
  if (p.after_many) pdl_wait();  // (it has nothing that this one reads)
}

// Joins the sequences that were cut: a warp per (KV head, query row) rescales the
// row's parts to their common maximum.
constexpr int kTailThreads = 256;
constexpr int kTailRows = kTailThreads / 32;

// Maximum and sum of a row over its parts [c0, c1] (lane i takes part c0 + i, + 32, ...).  part_f:
// this lane's last part, its index in part_ml and its factor 2^(m - M) (whole row when <= 32 parts).
struct RowParts {
  float M, Ls, f;
  int64_t w;
};
__device__ __forceinline__ RowParts row_parts(const PagedAttnParams& p, int64_t U, int C, int64_t s0, int c0, int c1,
                                              int kh, int r, int lane) {
  RowParts o{-INFINITY, 0.f, 0.f, 0};
  const int lanes = p.kv.hkv * p.row_blocks, ln = kh * p.row_blocks + r / p.block_rows;
  auto index = [&](int c) {
    return ((static_cast<int64_t>(c) * lanes + ln) * 2 + (few_first(U, C, c) >= s0 ? 0 : 1)) * p.block_rows +
           r % p.block_rows;
  };
  float2 v = make_float2(-INFINITY, 0.f);
  for (int c = c0 + lane; c <= c1; c += 32) {
    o.w = index(c);
    v = p.part_ml[o.w];
    o.M = fmaxf(o.M, v.x);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) o.M = fmaxf(o.M, __shfl_xor_sync(0xffffffffu, o.M, s));
  if (c1 - c0 < 32) {
    o.f = part_factor(v.x, o.M);
    o.Ls = v.y * o.f;
  } else {
    for (int c = c0 + lane; c <= c1; c += 32) {
      v = p.part_ml[index(c)];
      o.Ls += v.y * part_factor(v.x, o.M);
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) o.Ls += __shfl_xor_sync(0xffffffffu, o.Ls, s);
  return o;
}

template <int D>
__global__ void __launch_bounds__(kTailThreads) fna2_paged_few_join_kernel(const PagedAttnParams p) {
  const int kh = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int r = blockIdx.x * kTailRows + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  const PagedSeq sq = paged_seq(p.bd, b);
  const int units = few_units(p, sq);
  if (units == 0 || r >= sq.n * p.G) return;
  const int64_t U = p.prefix[p.bd.B], s0 = p.prefix[b];
  const int C = few_runs(p, U);
  const int c0 = few_run_of(U, C, s0), c1 = few_run_of(U, C, s0 + units - 1);
  if (c0 == c1) return;  // written by the attention kernel
  const RowParts o = row_parts(p, U, C, s0, c0, c1, kh, r, lane);
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int LD = D / 4;  // lanes that hold columns
  const int d = lane % LD * 4;
  for (int c = c0; c <= c1; c += 32) {
    // lane i holds part c + i (for more than 32 parts: found again)
    const RowParts q = c1 - c0 < 32 ? o : row_parts(p, U, C, s0, c, min(c1, c + 31), kh, r, lane);
    const float scale = c1 - c0 < 32 ? 1.f : part_factor(q.M, o.M);
    for (int i = 0; i <= min(31, c1 - c); ++i) {
      const int64_t w = __shfl_sync(0xffffffffu, q.w, i);
      const float f = __shfl_sync(0xffffffffu, q.f, i) * scale;
      const float4 a = *reinterpret_cast<const float4*>(p.part_acc + w * D + d);
      O.x += a.x * f, O.y += a.y * f, O.z += a.z * f, O.w += a.w * f;
    }
  }
  if (lane < LD) few_store<D>(p, sq.q0 + r % sq.n, kh * p.G + r / sq.n, d, o.M, o.Ls, O);
}

// Key weights of a call whose logits were kept: w[b, kh, j] += sum over the rows of
// 2^(x - LSE), 4 keys a thread.
constexpr int kLogitKeys = 4 * kTailThreads;

__global__ void __launch_bounds__(kTailThreads) fna2_paged_logit_weights_kernel(const PagedAttnParams p) {
  __shared__ float s_x[kLogitRows];
  pdl_wait();
  const int kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(p.bd, b);
  const int rows = sq.n * p.G, past = sq.len - sq.n, j = blockIdx.x * kLogitKeys + 4 * tid;
  if (static_cast<int>(blockIdx.x) * kLogitKeys >= sq.len || rows == 0) return;
  if (tid < rows) {
    const float v = p.lse2[static_cast<int64_t>(sq.q0 + tid % sq.n) * p.H + kh * p.G + tid / sq.n];
    s_x[tid] = v == -INFINITY ? INFINITY : v;  // a row without weight adds 0
  }
  __syncthreads();
  if (j >= sq.len) return;
  const float* x = p.logits + (static_cast<int64_t>(b) * p.kv.hkv + kh) * p.bd.max_q * p.G * p.logit_sr + j;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  int i = 0;  // new token of row r
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    // logits past what the row sees were not all written
    const int lim = p.causal ? min(sq.len, past + i + 1) : sq.len;
    i = i + 1 == sq.n ? 0 : i + 1;
    const float4 v = j < lim ? *reinterpret_cast<const float4*>(x + r * p.logit_sr) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] += j + k < lim ? ex2(vv[k] - s_x[r]) : 0.f;
  }
  float* kw = p.kw + b * p.kw_sb + kh * p.kw_sh + j;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (j + k < sq.len) kw[k] += w[k];
}

// Joins the tensor-core kernel's splits of one (token, query head), a warp each: rescale to the
// common max, O = acc / (l + 1e-6), LSE = m + log(l + 1e-6).
template <int D>
__global__ void __launch_bounds__(128) fna2_paged_many_join_kernel(const PagedAttnParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t th = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int64_t tok = th / p.H;
  const int h = static_cast<int>(th % p.H);
  if (tok >= p.bd.T) return;
  const int b = warp_seq_of(p.bd.cu, p.bd.B, tok, lane);
  if (b < 0) return;
  const PagedSeq sq = paged_seq(p.bd, b);
  const int ns = (sq.len + p.chunk_many - 1) / p.chunk_many;
  if (sq.n * p.G <= p.few_rows || ns <= 1) return;  // written by the attention kernels
  const float2* ml = p.ws_ml + th * p.ns;
  float M = -INFINITY;
  for (int s = 0; s < ns; ++s) M = fmaxf(M, ml[s].x);
  float Ls = 0.f;
  float O[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) O[i] = 0.f;
  for (int s = 0; s < ns; ++s) {
    const float2 v = ml[s];
    if (v.x == -INFINITY && v.y == 0.f) continue;  // no key of this split was seen, its output is not written
    const float f = part_factor(v.x, M);
    Ls += v.y * f;
    const float* a = p.ws_acc + (th * p.ns + s) * D + lane * (D / 32);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) O[i] += a[i] * f;
  }
  const float inv = 1.f / (Ls + kEps);
  __nv_bfloat16* o = p.out + tok * p.o_st + h * p.o_sh + lane * (D / 32);
#pragma unroll
  for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<uint32_t*>(o + i) = pack_bf16(O[i] * inv, O[i + 1] * inv);
  if (lane == 0 && p.lse) p.lse[h * p.lse_sh + tok] = (M + log2f(Ls + kEps)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <int D, int RW>
cudaError_t launch_paged_few_t(const PagedAttnParams& p, size_t smem, cudaStream_t stream) {
  auto kern = fna2_paged_few_kernel<D, RW>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed);
  if (e != cudaSuccess) return e;
  const unsigned grid = p.runs * p.kv.hkv * p.row_blocks;
  return launch_dependent(kern, grid, kFewThreads, smem, stream, p);
}

template <int D>
cudaError_t launch_paged_few_d(const PagedAttnParams& p, int RW, size_t smem, cudaStream_t stream) {
  return RW == 1   ? launch_paged_few_t<D, 1>(p, smem, stream)
         : RW == 2 ? launch_paged_few_t<D, 2>(p, smem, stream)
                   : launch_paged_few_t<D, 4>(p, smem, stream);
}

inline cudaError_t launch_paged_few(const PagedAttnParams& p, int D, int RW, size_t smem, cudaStream_t stream) {
  return D == 128 ? launch_paged_few_d<128>(p, RW, smem, stream) : launch_paged_few_d<64>(p, RW, smem, stream);
}

inline cudaError_t launch_paged_few_join(const PagedAttnParams& p, int D, cudaStream_t stream) {
  const int rows = std::min(p.bd.max_q * p.G, p.few_rows);
  const dim3 grid((rows + kTailRows - 1) / kTailRows, p.kv.hkv, p.bd.B);
  return launch_dependent(D == 128 ? fna2_paged_few_join_kernel<128> : fna2_paged_few_join_kernel<64>, grid, kTailThreads,
                          0, stream, p);
}

inline cudaError_t launch_logit_weights(const PagedAttnParams& p, cudaStream_t stream) {
  const dim3 grid((p.bd.max_k + kLogitKeys - 1) / kLogitKeys, p.kv.hkv, p.bd.B);
  return launch_dependent(fna2_paged_logit_weights_kernel, grid, kTailThreads, 0, stream, p);
}

inline cudaError_t launch_paged_many_join(const PagedAttnParams& p, int D, cudaStream_t stream) {
  const int64_t blocks = (static_cast<int64_t>(p.bd.T) * p.H + 3) / 4;
  return launch_dependent(D == 128 ? fna2_paged_many_join_kernel<128> : fna2_paged_many_join_kernel<64>,
                          static_cast<unsigned>(blocks), 128, 0, stream, p);
}

}  // namespace fna2
