// paged_attn.cu -- attention of one new token per sequence over a paged key-value cache.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,   p_t = 2^(log2(e) scale q_h . k_t - m),  m the running maximum
//
// Bound: HBM. Every key and value is read once and used by the q_heads / kv_heads queries that share
// it; per 16 tokens of one head that is 8 KB (bf16, head_dim 128) against 16 small matrix products.
//
// Work split. The unit is 16 or 32 tokens of one (sequence, key head). All units of a call, in the order
// (sequence, head, tokens), form one line that is cut into equal runs, one per CTA, and a CTA's run into one per
// warp (every (sequence, head) counts one unit more than it has, for its start and its end): no SM waits for a long sequence, whatever the lengths, and the lengths are read on the device, so a
// captured graph serves any of them. Each warp streams its run through its own ring in shared memory
// (cp.async, no barrier in the loop). What a warp has of a (sequence, head) that it shares with others is
// joined within the CTA through shared memory, and across CTAs by a second small kernel over partial
// results in the workspace; both joins add in the line's order, so results do not depend on timing. Few short sequences go
// without a line: a CTA each per key head ("solo").
//
// Matrix products are m16n8k16 with the TOKENS as the 16 rows and up to eight query heads as the eight
// columns (a GQA group of four or eight wastes half or nothing; queries as rows would waste three quarters
// and need twice the accumulators). S^T = K Q^T comes out with tokens in rows; P enters the second product,
// O^T = V^T P^T, as its B operand, which wants the 8 x 8 blocks transposed: one movmatrix each.
//
// 8-bit caches multiply the codes, not the values. A byte c with a zero byte above it IS the fp16 number
// c 2^-24 (a subnormal), so a pair of operands costs one byte permute. With k = s c + b, g: groups of 64,
//   q . k = sum_g s_g (q . c)_g + b_g sum_g q
//   o     = sum_t p'_tg c - 128 sum_t p'_tg + sum_t p_t (b_tg + 128 s_tg),   p'_tg = p_t s_tg rounded to fp16
// and scales and biases act on 16 x 8 scores instead of 16 x head_dim values. The middle term of o (one
// product with a constant operand per group) takes the codes' mean out of the rounding of p' and, subtracted
// unit by unit, out of the sums. q is scaled by a power of two per head to fill fp16's range (exact up to 2^-39 of
// the head's largest value); p s is taken relative to a running power of two above every scale, times 2^15,
// which keeps its rounding at 2^-11 relative down to 2^-29.
// In a bf16 cache p is rounded to bf16 (2^-8) and the sum of weights adds the rounded p, so the
// weights still sum to one.
#include "vpq_kv.cuh"
#include "vpq_sm100.cuh"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace vpq {

namespace {

constexpr float kNegInf = -__builtin_huge_valf();

// What the joining kernel has to know of a CTA: the (sequence, head) that begins in its run and goes on in
// the next CTA's (its first query head, and how many), where its partial result is (0: the run's first, 1), and
// the last CTA that has a part.
struct CtaHead {
  int b, h, ncol_slot, last;  // ncol << 1 | slot; last -1: none
};

struct AttnArgs {
  KvView kv;
  const uint8_t* q;
  uint8_t* out;
  uint32_t* status;              // index reports
  int64_t q_stride, out_stride;  // bytes
  const int32_t* page_table;
  const int32_t* seq_lens;
  int64_t table_stride;
  CtaHead* heads;    // workspace: one per CTA
  float* ml;         // [CTA][2][cols][2]: maximum and sum of a partial result
  float* part;       // [CTA][2][cols][D]
  float* scratch;    // [CTA][warp][cols][D]: a warp's first partial result, if another run follows it; null: in
                     // shared memory behind the rings
  int batch, max_pages, window;
  int group;         // query heads of a key head
  int cols;          // query heads a unit serves (a column block): min(group, 8 NT)
  int blocks;        // column blocks of a key head
  int hk;            // kv_heads * blocks
  uint32_t cta_rcp;  // 2^32 / CTAs, rounded up: a quotient may come out one too large, which is as good a cut
  bool solo;         // a CTA per (sequence, column block), and no second kernel
  bool dense;        // rows of a page's head lie back to back
  bool few;          // at most 32 sequences, and few enough units for 32-bit sums
  float scale_log2;
  int stage_bytes, ring_bytes;  // shared memory: a stage, a warp's ring
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(live ? BYTES : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <bool HALF>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HALF) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lo16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// Bytes 0, 1 of w (HI: 2, 3), each with a zero byte above: the fp16 numbers c 2^-24.
template <bool HI>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
  return __byte_perm(w, 0u, HI ? 0x4342 : 0x4140);
}
// Quotients of numbers that nearly always fit 32 bits (a 64-bit division costs five times as much).
__device__ __forceinline__ int64_t div_u(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// The scale pairs of a row.
template <int G>
__device__ __forceinline__ void lds_pairs(uint32_t (&p)[G], uint32_t a) {
  if (G == 1) {
    p[0] = lds32(a);
  } else if (G == 2) {
    const uint2 w = lds64(a);
    p[0] = w.x, p[G > 1 ? 1 : 0] = w.y;
  } else {
    const uint4 w = lds128(a);
    p[0] = w.x, p[G > 1 ? 1 : 0] = w.y, p[G > 2 ? 2 : 0] = w.z, p[G > 3 ? 3 : 0] = w.w;
  }
}
// Where value d of column col lies in its row of a warp's partial result: the 32 lanes that store
// together fall into 32 banks.
template <int BITS, bool HALF>
__device__ __forceinline__ int entry_at(int col, int d) {
  const int t = (HALF ? col : col >> 1) & 3;  // the lanes of a quad
  return BITS == 16 ? d ^ (t << 3) : d ^ t ^ ((d >> 3) & 4);
}
// The factor that takes a partial result (maximum m, sum l) to the joint maximum; one without a live token
// counts nothing, unless it holds a NaN.
__device__ __forceinline__ float weight_of(float m, float l, float joint) {
  return m == kNegInf ? (l == 0.0f ? 0.0f : 1.0f) : ex2(m - joint);
}

// Tokens of sequence b that count: [start, len), len cut to what the table can name.
__device__ __forceinline__ void token_range(const AttnArgs& A, int b, int& start, int& len) {
  int n = __ldg(A.seq_lens + b);
  const int64_t cap = (int64_t)A.max_pages * A.kv.page_size;
  if ((int64_t)n > cap) { n = (int)cap; }
  len = n > 0 ? n : 0;
  start = (A.window > 0 && len > A.window) ? len - A.window : 0;
}
template <int U>
__device__ __forceinline__ int units_of(int start, int len) {
  return len > start ? (len + U - 1) / U - start / U : 0;
}
// Its length on the line, per head: one place for the start and the end of a (sequence, head), then its units.
template <int U>
__device__ __forceinline__ int span_of(int start, int len) {
  const int n = units_of<U>(start, len);
  return n > 0 ? n + 1 : 0;
}

// Where 16-byte chunk c of row `row` lies in a K or V tile: chunk c ^ swz(row). 16 bits: the eight rows that an
// ldmatrix reads fall into eight bank groups. 8 bits: see the loads in the loop.
template <int D, int BITS>
__device__ __forceinline__ constexpr int swz_k(int row) {
  return BITS == 16 ? row & 7 : (D >= 128 ? (row & 1) << 2 : 0);
}
template <int D, int BITS>
__device__ __forceinline__ constexpr int swz_v(int row) {
  return BITS == 16 ? row & 7 : (D >= 128 ? row & 6 : row & 2);
}

// What a unit in flight is: written by lane 0 with its copies, read when its turn comes.
struct alignas(16) UnitMeta {
  int b, h;       // sequence; first query head of the column block
  int bits;       // live rows [lo, hi): lo | hi << 8, flags << 16, columns << 24
  int rest;       // units of this (sequence, head) behind this one
};
enum : int { kFirst = 1 << 16, kLast = 2 << 16, kSegBegin = 4 << 16 };

// A partial result of a warp. It has room for two: of its first run, if others follow, in the workspace,
// and of its last run, over its ring.
struct EntryHead {
  int b, h;     // b -1: none
  int begins;   // from the first token on
  int rest;     // as UnitMeta, of its last unit
  int leads;    // the first of the CTA's line
  int ncol;
  float m[16], l[16];
};

template <int D, int BITS, int NT, bool HALF, int TM, int kWarps, int STAGES>
__global__ void __launch_bounds__(kWarps * 32, 1) paged_attn_kernel(const AttnArgs A) {
  constexpr int kUnit = 16 * TM;
  constexpr int kRow = D * BITS / 8;
  constexpr int kTile = kUnit * kRow;
  constexpr int G = D / kKvGroup;
  constexpr int kPair = BITS == 8 ? G * 4 : 0;  // scale pairs of a row
  constexpr int kPairs = kUnit * kPair;
  constexpr int MT = D / 16;  // 16-row blocks of O^T
  // Up to four query heads (HALF) sit in every other column, so that a lane of a product has one live column and not
  // two (or none): half the work between the two products.
  static_assert(!HALF || NT == 1, "four columns fit one product");
  constexpr int CN = HALF ? 1 : 2;  // live columns of a lane
  constexpr int kNone = 1 << 20;

  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_excl[kWarps * 32];
  __shared__ int2 s_range[kWarps * 32];
  __shared__ int64_t s_wsum[kWarps];
  __shared__ UnitMeta s_meta[kWarps][STAGES];
  __shared__ EntryHead s_entry[kWarps * 2];
  __shared__ float s_f[kWarps * 2][16], s_fl[kWarps * 2][16];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, t = lane & 3;
  auto col_of = [&](int n, int c) { return HALF ? t : n * 8 + 2 * t + c; };        // of this lane's accumulators
  auto col_in = [&](int n) { return HALF ? ((r & 1) ? kNone : r >> 1) : n * 8 + r; };  // of its operands

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run of the line of units. Up to 32 sequences: every warp looks at all of them; more: a
  // thread at a few neighbouring ones each.
  if (lane < 2) { s_entry[warp * 2 + lane].b = -1; }
  int left = 0;  // places of the line that this warp has yet to request
  int todo = 0;  // units requested and not yet computed
  int64_t cta0 = 0, cta1 = 0, per_cta = 1;
  // ---- the loader's place in the line
  int lb = 0, lh = 0, lkv = 0, lblk = 0, ltile = 0, ltile0 = 0, ltile_end = 0, lstart = 0, llen = 0;
  int pg = 0, off = 0;     // page-table column and token offset in the page
  bool fresh = true;       // the next unit begins a (sequence, head) for this warp
  int page[TM];            // page numbers of the next unit, fetched one unit ahead; -1: none
  auto enter = [&]() {     // to the first token of unit ltile
    const uint32_t at = (uint32_t)ltile * kUnit;
    pg = (int)(A.kv.page_shift >= 0 ? at >> A.kv.page_shift : at / (uint32_t)A.kv.page_size);
    off = (int)(at - (uint32_t)pg * (uint32_t)A.kv.page_size);
  };
  auto fetch_pages = [&]() {
    int c = pg, o = off;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int first = ltile * kUnit + 16 * i;
      // entries of pages without a live token are not read
      page[i] = (first < llen && first + 16 > lstart) ? __ldg(A.page_table + (int64_t)lb * A.table_stride + c) : -1;
      o += 16;
      if (o == A.kv.page_size) { o = 0, ++c; }
    }
  };
  if (A.solo) {
    // all of one (sequence, column block), a warp having a stretch of its units
    lb = (int)(blockIdx.x / (uint32_t)A.hk), lh = (int)(blockIdx.x - (uint32_t)lb * (uint32_t)A.hk);
    lkv = A.blocks == 1 ? lh : lh / A.blocks;
    lblk = lh - lkv * A.blocks;
    token_range(A, lb, lstart, llen);
    if (tid == 0 && lh == 0 && __ldg(A.seq_lens + lb) > llen) { atomicOr(A.status, kBadLength); }
    const int n = units_of<kUnit>(lstart, llen);
    if (n == 0) {  // no token: zeros
      const int h0 = lkv * A.group + lblk * A.cols, ncol = min(A.cols, A.group - lblk * A.cols);
      uint4* row = reinterpret_cast<uint4*>(A.out + (int64_t)lb * A.out_stride + (int64_t)h0 * (D * 2));
      for (int i = tid; i < ncol * (D / 8); i += kWarps * 32) { row[i] = make_uint4(0, 0, 0, 0); }
      return;
    }
    const int per_warp = (n + kWarps - 1) / kWarps;
    left = max(0, min(per_warp, n - warp * per_warp));
    ltile0 = lstart / kUnit;
    ltile_end = ltile0 + n;
    ltile = ltile0 + warp * per_warp;
    if (left > 0) {
      enter();
      fetch_pages();
    }
  } else {
    if (tid == 0) { A.heads[blockIdx.x].last = -1; }
    const int cpt = A.few ? 1 : (A.batch + kWarps * 32 - 1) / (kWarps * 32);
    const int me = A.few ? lane : tid;
    const int b_lo = min(me * cpt, A.batch), b_hi = min(b_lo + cpt, A.batch);
    int64_t mine = 0;
    int2 seen = make_int2(0, 0);  // token range of the last of them
    for (int b = b_lo; b < b_hi; ++b) {
      token_range(A, b, seen.x, seen.y);
      mine += span_of<kUnit>(seen.x, seen.y);
      if (blockIdx.x == 0 && __ldg(A.seq_lens + b) > seen.y) { atomicOr(A.status, kBadLength); }
    }
    int64_t excl, total;  // places (of one head) before the first of them, and of all
    if (A.few) {
      int incl = (int)mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) { incl += o; }
      }
      excl = incl - (int)mine;
      total = __shfl_sync(0xffffffffu, incl, 31);
    } else {
      int64_t incl = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) { incl += o; }
      }
      if (lane == 31) { s_wsum[warp] = incl; }
      __syncthreads();
      excl = incl - mine;
      total = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) { excl += s_wsum[w]; }
        total += s_wsum[w];
      }
      s_excl[tid] = excl;
      s_range[tid] = seen;
      __syncthreads();
    }
    const int64_t places = total * A.hk;
    // (32-bit numbers by the reciprocal that the host has made of the number of CTAs)
    per_cta = (places + gridDim.x) >> 31 == 0 ? (int64_t)__umulhi((uint32_t)places + gridDim.x - 1, A.cta_rcp)
                                                      : (places + gridDim.x - 1) / gridDim.x;
    per_cta = per_cta > kWarps ? per_cta : kWarps;
    cta0 = (int64_t)blockIdx.x * per_cta;
    if (cta0 >= places) { return; }  // the whole CTA
    cta1 = cta0 + per_cta < places ? cta0 + per_cta : places;
    const int64_t per_warp = (cta1 - cta0 + kWarps - 1) / kWarps;
    const int64_t u0 = cta0 + warp * per_warp;
    const int64_t u1 = u0 + per_warp < cta1 ? u0 + per_warp : cta1;
    left = u0 < u1 ? (int)(u1 - u0) : 0;
    if (left > 0) {
      // who looked at u0's sequence: the last whose sequences begin at or before it
      int64_t at;
      if (A.few) {
        lb = 31 - __clz(__ballot_sync(0xffffffffu, excl * A.hk <= u0));
        at = __shfl_sync(0xffffffffu, excl, lb);
        lstart = __shfl_sync(0xffffffffu, seen.x, lb), llen = __shfl_sync(0xffffffffu, seen.y, lb);
      } else {
        int64_t upto = 0;
        int tw = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (upto * A.hk <= u0) { tw = w; }
          upto += s_wsum[w];
        }
        const int64_t ex = s_excl[tw * 32 + lane];
        const int tl = 31 - __clz(__ballot_sync(0xffffffffu, ex * A.hk <= u0));
        at = __shfl_sync(0xffffffffu, ex, tl);
        lb = (tw * 32 + tl) * cpt;
        if (cpt == 1) {
          lstart = s_range[tw * 32 + tl].x, llen = s_range[tw * 32 + tl].y;
        } else {
          for (;; ++lb) {
            token_range(A, lb, lstart, llen);
            const int n = span_of<kUnit>(lstart, llen);
            if ((at + n) * A.hk > u0) { break; }
            at += n;
          }
        }
      }
      ltile0 = lstart / kUnit;
      ltile_end = ltile0 + units_of<kUnit>(lstart, llen);
      const int64_t in_seq = u0 - at * A.hk;
      const int span = ltile_end - ltile0 + 1;
      lh = (int)div_u(in_seq, span);
      const int place = (int)(in_seq - (int64_t)lh * span);
      ltile = ltile0 + (place > 0 ? place - 1 : 0);
      if (place == 0) { --left; }
      lkv = A.blocks == 1 ? lh : lh / A.blocks;
      lblk = lh - lkv * A.blocks;
      if (left > 0) {
        enter();
        fetch_pages();
      }
    }
  }

  uint8_t* ring = smem + warp * A.ring_bytes;
  float* scratch0 = A.scratch ? A.scratch + (int64_t)blockIdx.x * kWarps * (A.cols * D)
                              : reinterpret_cast<float*>(smem + kWarps * A.ring_bytes);
  const uint32_t ring_s = smem_u32(ring);
  constexpr int CH = kRow / 16;                      // 16-byte chunks of a row
  constexpr int kRowsPer = CH < 32 ? 32 / CH : 1;    // rows that one round of the warp's copies covers
  constexpr int kRounds = 16 * CH / 32;
  const int crow = CH < 32 ? lane / CH : 0, cch = lane % CH;
  // A lane's place in a tile; the swizzles of the lane's row and of a round's act on different bits.
  const uint32_t lane_k = crow * kRow + ((cch ^ swz_k<D, BITS>(crow)) << 4);
  const uint32_t lane_v = crow * kRow + ((cch ^ swz_v<D, BITS>(crow)) << 4);
  const int64_t v_minus_k = A.kv.v - A.kv.k;
  const uint8_t *head_k = nullptr, *head_s = nullptr;  // this lane's row of page 0 of the current key head
  auto enter_head = [&]() {
    head_k = A.kv.k + (uint64_t)(uint32_t)lkv * A.kv.head_bytes + (uint64_t)(uint32_t)crow * A.kv.token_bytes + cch * 16;
    if (BITS == 8) {
      head_s = (lane < 16 ? A.kv.ks : A.kv.vs) + (uint64_t)(uint32_t)lkv * A.kv.shead_bytes +
               (uint64_t)(uint32_t)(lane & 15) * A.kv.stoken_bytes;
    }
  };
  enter_head();

  // Requests the next unit into stage `st`; commits a group in any case.
  auto request = [&](int st) {
    if (left > 0) {
      int lo = lstart - ltile * kUnit;
      lo = lo > 0 ? lo : 0;
      int hi = llen - ltile * kUnit;
      hi = hi < kUnit ? hi : kUnit;
      const uint32_t dst = ring_s + st * A.stage_bytes;
      bool plain = A.dense && lo == 0 && hi == kUnit;
#pragma unroll
      for (int i = 0; i < TM; ++i) { plain = plain && (uint32_t)page[i] < (uint32_t)A.kv.num_pages; }
      int bad = 0;
      if (plain) {
        // every row lives, rows lie back to back: nothing but copies at constant distances
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const uint8_t* kp = head_k + (uint64_t)(uint32_t)page[i] * A.kv.page_bytes + off * kRow;
          const uint8_t* vp = kp + v_minus_k;
#pragma unroll
          for (int j = 0; j < kRounds; ++j) {
            constexpr int kStep = kRowsPer;
            cp_async16(dst + (lane_k ^ (swz_k<D, BITS>(j * kStep) << 4)) + (16 * i + j * kStep) * kRow, kp + j * kStep * kRow);
            cp_async16(dst + (lane_v ^ (swz_v<D, BITS>(j * kStep) << 4)) + kTile + (16 * i + j * kStep) * kRow,
                       vp + j * kStep * kRow);
          }
          if (BITS == 8) {
            cp_async_small<kPair ? kPair : 4>(dst + 2 * kTile + (lane < 16 ? 0 : kPairs) + (16 * i + (lane & 15)) * kPair,
                                              head_s + (uint64_t)(uint32_t)page[i] * A.kv.spage_bytes + off * kPair, true);
          }
          off += 16;
          if (off == A.kv.page_size) { off = 0, ++pg; }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < TM; ++i) {
          const int pi = TM == 2 && i == 1 ? page[TM - 1] : page[0];
          const bool ok = (uint32_t)pi < (uint32_t)A.kv.num_pages;
          // A page without live tokens, or none: rows of zeros. Dead rows of a page become zeros too: whatever
          // they hold, their weight 0 has to add 0.
          const int rlo = ok ? lo - 16 * i : 16, rhi = ok ? hi - 16 * i : 0;
          if (!ok && lo < 16 * i + 16 && hi > 16 * i) { bad |= 1 << i; }
          const uint64_t pp = ok ? (uint32_t)pi : 0;
          const uint8_t* kp = head_k + pp * A.kv.page_bytes + (uint64_t)(uint32_t)off * A.kv.token_bytes;
#pragma unroll
          for (int j = 0; j < kRounds; ++j) {
            const int row = crow + j * kRowsPer;
            const bool live = row >= rlo && row < rhi;
            const uint8_t* kr = kp + (uint64_t)(j * kRowsPer) * A.kv.token_bytes;
            const uint32_t to = dst + (16 * i + j * kRowsPer) * kRow;
            cp_async16(to + (lane_k ^ (swz_k<D, BITS>(j * kRowsPer) << 4)), kr, live);
            cp_async16(to + kTile + (lane_v ^ (swz_v<D, BITS>(j * kRowsPer) << 4)), kr + v_minus_k, live);
          }
          if (BITS == 8) {
            const int row = lane & 15;
            cp_async_small<kPair ? kPair : 4>(dst + 2 * kTile + (lane < 16 ? 0 : kPairs) + (16 * i + row) * kPair,
                                              head_s + pp * A.kv.spage_bytes + (uint64_t)(uint32_t)off * A.kv.stoken_bytes,
                                              row >= rlo && row < rhi);
          }
          off += 16;
          if (off == A.kv.page_size) { off = 0, ++pg; }
        }
      }
      if (bad) {  // a page outside the cache holds no tokens: the live rows shrink to what is left
        if (lane == 0) { atomicOr(A.status, kBadPage); }
        if (TM == 1 || bad == 3) {
          lo = hi = 0;
        } else if (bad == 1) {
          lo = min(max(lo, 16), hi);
        } else {
          hi = max(min(hi, 16), lo);
        }
      }
      const int h0 = lkv * A.group + lblk * A.cols;
      const int ncol = min(A.cols, A.group - lblk * A.cols);
      if (fresh) {
        const uint8_t* qp = A.q + (int64_t)lb * A.q_stride + (int64_t)h0 * (D * 2);
        for (int i = lane; i < ncol * (D / 8); i += 32) { cp_async16(dst + 2 * kTile + 2 * kPairs + i * 16, qp + i * 16); }
      }
      const int rest = ltile_end - 1 - ltile;
      if (lane == 0) {
        s_meta[warp][st] = {lb, h0,
                            lo | (hi << 8) | (ncol << 24) | (fresh ? kFirst : 0) | ((left == 1 || rest == 0) ? kLast : 0) |
                                (ltile == ltile0 ? kSegBegin : 0),
                            rest};
      }
      ++todo;
      --left;
      fresh = false;
      ++ltile;
      if (left > 0 && rest == 0) { --left; }
      if (left > 0) {
        if (rest == 0) {
          fresh = true;
          ++lh;
          if (++lblk == A.blocks) { lblk = 0, ++lkv; }
          if (lh == A.hk) {
            lh = lkv = lblk = 0;
            do {
              ++lb;
              token_range(A, lb, lstart, llen);
            } while (units_of<kUnit>(lstart, llen) == 0);
            ltile0 = lstart / kUnit;
            ltile_end = ltile0 + units_of<kUnit>(lstart, llen);
          }
          ltile = ltile0;
          enter();
          enter_head();
        }
        fetch_pages();
      }
    }
    cp_commit();
  };

  float o_acc[NT][MT][4];
  float m_run[NT][CN], l_run[NT][CN];
  float o_bias[NT][G][CN], q_sum[NT][G][CN], q_mul[NT][CN];  // 8 bits
  uint32_t qf[NT][D / 16][2];
  int sigma = -100;      // 8 bits: exponent of the power of two above every value scale so far
  bool run_begins = false, first_run = true;

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) { request(s); }

  for (int st = 0; todo > 0; --todo) {
    cp_wait<STAGES - 2>();
    __syncwarp();  // the stage's copies and its record are visible; the stage before is free
    const UnitMeta U = s_meta[warp][st];
    request(st == 0 ? STAGES - 1 : st - 1);
    const uint32_t kt = ring_s + st * A.stage_bytes, vt = kt + kTile, ksc = vt + kTile, vsc = ksc + kPairs,
                   qt = vsc + kPairs;

    if (U.bits & kFirst) {
      const int ncol = U.bits >> 24;
      run_begins = (U.bits & kSegBegin) != 0;
      sigma = -100;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < CN; ++c) { m_run[n][c] = kNegInf, l_run[n][c] = 0.0f; }
#pragma unroll
        for (int i = 0; i < MT; ++i) { o_acc[n][i][0] = o_acc[n][i][1] = o_acc[n][i][2] = o_acc[n][i][3] = 0.0f; }
        const bool live = col_in(n) < ncol;
        const uint32_t qrow = qt + (live ? col_in(n) : 0) * (D * 2);
        if (BITS == 16) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            qf[n][k][0] = live ? lds32(qrow + k * 32 + t * 4) : 0u;
            qf[n][k][1] = live ? lds32(qrow + k * 32 + 16 + t * 4) : 0u;
          }
        } else {
          // lane t of a quad holds values 64 g + 16 t + 0..15 of its column
          float top = 0.0f, sum[G];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            sum[g] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 w4 = live ? lds128(qrow + g * 128 + t * 32 + i * 16) : make_uint4(0, 0, 0, 0);
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                qf[n][g * 4 + i * 2 + e / 2][e & 1] = w[e];
                sum[g] += lo16(w[e]) + hi16(w[e]);
                top = fmaxf(top, fmaxf(fabsf(lo16(w[e])), fabsf(hi16(w[e]))));
              }
            }
            sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
            sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // largest value to [2^14, 2^15); a row of zeros, NaN or infinities keeps its values' meaning
          int e = (int)(__float_as_uint(top) >> 23) - 127;
          e = min(max(e, -100), 127);
          const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
          const float down = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
          // a code's 2^24, the power of two and the scale in an order in which nothing but their product can overflow
          const float mul = e > 100 ? down * A.scale_log2 * 16777216.0f : down * 16777216.0f * A.scale_log2;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
#pragma unroll
            for (int i = 0; i < 2; ++i) { qf[n][k][i] = pack_f16x2(lo16(qf[n][k][i]) * up, hi16(qf[n][k][i]) * up); }
          }
#pragma unroll
          for (int c = 0; c < CN; ++c) {  // the same for the columns of this lane's scores
            q_mul[n][c] = __shfl_sync(0xffffffffu, mul, (2 * t + c) * 4);
#pragma unroll
            for (int g = 0; g < G; ++g) {
              q_sum[n][g][c] = __shfl_sync(0xffffffffu, sum[g], (2 * t + c) * 4) * A.scale_log2;
              o_bias[n][g][c] = 0.0f;
            }
          }
        }
      }
    }

    // ---- scores times log2(e) scale: rows 16 i + r, 16 i + r + 8 of the unit, columns 2t, 2t + 1
    float s[TM][NT][4];
    if (BITS == 16) {
      const int row = (lane & 7) + (lane & 8), ch = lane >> 4;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) { s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.0f; }
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          uint32_t a[4];
          ldsm4(a, kt + (16 * i + row) * kRow + ((2 * k + ch) ^ swz_k<D, BITS>(row)) * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) { mma<false>(s[i][n], a, qf[n][k][0], qf[n][k][1]); }
        }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; e += 3 - CN) { s[i][n][e] *= A.scale_log2; }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        uint32_t p0[G], p1[G];
        lds_pairs<G>(p0, ksc + (16 * i + r) * kPair);
        lds_pairs<G>(p1, ksc + (16 * i + r + 8) * kPair);
        float bias[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; e += 3 - CN) { s[i][n][e] = bias[n][e] = 0.0f; }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          // a lane's 16 codes feed four k steps: the k order is permuted the same way in q
          const uint4 x = lds128(kt + (16 * i + r) * kRow + ((4 * g + t) ^ swz_k<D, BITS>(r)) * 16);
          const uint4 y = lds128(kt + (16 * i + r + 8) * kRow + ((4 * g + t) ^ swz_k<D, BITS>(r + 8)) * 16);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
          float c[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) { c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f; }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t a[4] = {codes<false>(xs[u]), codes<false>(ys[u]), codes<true>(xs[u]), codes<true>(ys[u])};
#pragma unroll
            for (int n = 0; n < NT; ++n) { mma<true>(c[n], a, qf[n][g * 4 + u][0], qf[n][g * 4 + u][1]); }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; e += 3 - CN) {
              const uint32_t p = e < 2 ? p0[g] : p1[g];
              s[i][n][e] = __fmaf_rn(c[n][e], lo16(p), s[i][n][e]);
              bias[n][e] = __fmaf_rn(hi16(p), q_sum[n][g][e & (CN - 1)], bias[n][e]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; e += 3 - CN) { s[i][n][e] = __fmaf_rn(s[i][n][e], q_mul[n][e & (CN - 1)], bias[n][e]); }
        }
      }
    }
    const int lo = U.bits & 0xff, hi = (U.bits >> 8) & 0xff;
    if (lo > 0 || hi < kUnit) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; e += 3 - CN) {
            const int row = 16 * i + r + (e < 2 ? 0 : 8);
            s[i][n][e] = row >= lo && row < hi ? s[i][n][e] : kNegInf;
          }
        }
      }
    }
    bool grows = false;
    float m_new[NT][CN];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        float x = fmaxf(s[0][n][c], s[0][n][2 + c]);
#pragma unroll
        for (int i = 1; i < TM; ++i) { x = fmaxf(x, fmaxf(s[i][n][c], s[i][n][2 + c])); }
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        m_new[n][c] = fmaxf(m_run[n][c], x);
        grows |= m_new[n][c] > m_run[n][c];
      }
    }
    // 8 bits: this lane's value pairs, and the power of two above their scales
    uint32_t vp[TM][2][G];
    float rescale = 1.0f, up = 1.0f;
    if (BITS == 8) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds_pairs<G>(vp[i][h], vsc + (16 * i + r + 8 * h) * kPair);
#pragma unroll
          for (int g = 0; g < G; ++g) { top = max(top, vp[i][h][g] & 0x7fffu); }
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (top >= 0x7f80u) {  // a NaN or an infinity spoils its own group's values; the others' rounding does not go by it
        top = 0;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const uint32_t x = vp[i][h][g] & 0x7fffu;
              top = max(top, x < 0x7f80u ? x : 0u);
            }
          }
        }
        top = __reduce_max_sync(0xffffffffu, top);
      }
      const int e = (int)(top >> 7) - 126;  // every scale that is a number is below 2^e
      if (e > sigma) {
        grows = true;
        rescale = ex2((float)(sigma - e));
        sigma = e;
      }
      up = __uint_as_float((uint32_t)(15 - sigma + 127) << 23);
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < CN; ++c) {
          const float f = m_new[n][c] > m_run[n][c] ? ex2(m_run[n][c] - m_new[n][c]) : 1.0f;
          m_run[n][c] = m_new[n][c];
          l_run[n][c] *= f;
          const float fo = f * rescale;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o_acc[n][i][c] *= fo;
            o_acc[n][i][2 + c] *= fo;
          }
          if (BITS == 8) {
#pragma unroll
            for (int g = 0; g < G; ++g) { o_bias[n][g][c] *= f; }
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        const float m = m_run[n][c] == kNegInf ? 0.0f : m_run[n][c];  // no live token yet: 2^-inf, not NaN
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          s[i][n][c] = ex2(s[i][n][c] - m);
          s[i][n][2 + c] = ex2(s[i][n][2 + c] - m);
        }
      }
    }

    // ---- O^T += V^T P^T
    if (BITS == 16) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        uint32_t b[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = pack_bf16x2(s[i][n][2 * h], HALF ? 0.0f : s[i][n][2 * h + 1]);
            l_run[n][0] += lo16(w);
            if (!HALF) { l_run[n][CN - 1] += hi16(w); }
            b[n][h] = movm(w);
          }
        }
        const int row = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < MT; ++k) {
          uint32_t a[4];
          ldsm4t(a, vt + (16 * i + row) * kRow + ((2 * k + ch) ^ swz_v<D, BITS>(row)) * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) { mma<false>(o_acc[n][k], a, b[n][0], b[n][1]); }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int c = 0; c < CN; ++c) { l_run[n][c] += s[i][n][c] + s[i][n][2 + c]; }
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t b[TM][NT][2], x[TM][2][4];
        float mean[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) { mean[n][0] = mean[n][1] = mean[n][2] = mean[n][3] = 0.0f; }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float sc = lo16(vp[i][h][g]), f = sc * up, bb = __fmaf_rn(128.0f, sc, hi16(vp[i][h][g]));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              b[i][n][h] = movm(pack_f16x2(s[i][n][2 * h] * f, HALF ? 0.0f : s[i][n][2 * h + 1] * f));
#pragma unroll
              for (int c = 0; c < CN; ++c) { o_bias[n][g][c] = __fmaf_rn(s[i][n][2 * h + c], bb, o_bias[n][g][c]); }
            }
          }
          const uint32_t k128[4] = {0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u};  // the code 128
#pragma unroll
          for (int n = 0; n < NT; ++n) { mma<true>(mean[n], k128, b[i][n][0], b[i][n][1]); }
          // codes 64 g + 8 r + 0..7 of tokens 2t, 2t + 1, 2t + 8, 2t + 9. A row's eight lanes of equal t read 64
          // bytes; the swizzle puts the four token pairs of a half warp into different banks.
          uint2 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = 2 * t + (j & 1) + (j >> 1) * 8;
            w[j] = lds64(vt + (16 * i + row) * kRow + ((4 * g + (r >> 1)) ^ swz_v<D, BITS>(row)) * 16 + (r & 1) * 8);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // per token pair: values 0|1, 2|3, 4|5, 6|7 as bytes (even token, odd token, ...)
            x[i][h][0] = __byte_perm(w[2 * h].x, w[2 * h + 1].x, 0x5140);
            x[i][h][1] = __byte_perm(w[2 * h].x, w[2 * h + 1].x, 0x7362);
            x[i][h][2] = __byte_perm(w[2 * h].y, w[2 * h + 1].y, 0x5140);
            x[i][h][3] = __byte_perm(w[2 * h].y, w[2 * h + 1].y, 0x7362);
          }
        }
        // The products of a unit start from zero, and what is added up is their distance from the mean's: the sums
        // over a long sequence would otherwise be 128 times the weights, next to which the product unit cuts off
        // what the values differ by (measured at 131072 equal weights: a third of the result).
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // rows r, r + 8 of this block: values 64 g + 8 r + 2 k, + 1
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              const uint32_t a[4] = {codes<false>(x[i][0][k]), codes<true>(x[i][0][k]), codes<false>(x[i][1][k]),
                                     codes<true>(x[i][1][k])};
              mma<true>(c, a, b[i][n][0], b[i][n][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; e += 3 - CN) { o_acc[n][g * 4 + k][e] += c[e] - mean[n][e & 1]; }
          }
        }
      }
    }

    // ---- the warp's part of a (sequence, head) is complete
    if (U.bits & kLast) {
      const int ncol = U.bits >> 24;
      const float o_mul = BITS == 8 ? __uint_as_float((uint32_t)(sigma - 15 + 127) << 23) : 1.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < CN; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            l_run[n][c] += __shfl_xor_sync(0xffffffffu, l_run[n][c], d);
            if (BITS == 8) {
#pragma unroll
              for (int g = 0; g < G; ++g) { o_bias[n][g][c] += __shfl_xor_sync(0xffffffffu, o_bias[n][g][c], d); }
            }
          }
        }
        if (BITS == 8) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int e = 0; e < 4; e += 3 - CN) {
              o_acc[n][i][e] = __fmaf_rn(o_acc[n][i][e] * 16777216.0f, o_mul, o_bias[n][i / 4][e & (CN - 1)]);
            }
          }
        }
      }
      if (run_begins && U.rest == 0) {
        uint8_t* op = A.out + (int64_t)U.b * A.out_stride + (int64_t)U.h * (D * 2);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // a sum of 0: no live token (a NaN stays one)
          float inv[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) { inv[c] = c >= CN || l_run[n][c % CN] == 0.0f ? 0.0f : 1.0f / l_run[n][c % CN]; }
          if (BITS == 16) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w = movm(pack_bf16x2(o_acc[n][i][2 * h] * inv[0], HALF ? 0.0f : o_acc[n][i][2 * h + 1] * inv[1]));
                if (col_in(n) < ncol) {
                  *reinterpret_cast<uint32_t*>(op + col_in(n) * (D * 2) + (16 * i + 8 * h + 2 * t) * 2) = w;
                }
              }
            }
          } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
              for (int c = 0; c < CN; ++c) {
                const int col = col_of(n, c);
                uint4 y;
                y.x = pack_bf16x2(o_acc[n][g * 4][c] * inv[c], o_acc[n][g * 4][2 + c] * inv[c]);
                y.y = pack_bf16x2(o_acc[n][g * 4 + 1][c] * inv[c], o_acc[n][g * 4 + 1][2 + c] * inv[c]);
                y.z = pack_bf16x2(o_acc[n][g * 4 + 2][c] * inv[c], o_acc[n][g * 4 + 2][2 + c] * inv[c]);
                y.w = pack_bf16x2(o_acc[n][g * 4 + 3][c] * inv[c], o_acc[n][g * 4 + 3][2 + c] * inv[c]);
                if (col < ncol) { *reinterpret_cast<uint4*>(op + col * (D * 2) + (64 * g + 8 * r) * 2) = y; }
              }
            }
          }
        }
      } else {
        const bool done = todo == 1;
        EntryHead& H = s_entry[warp * 2 + done];
        float* to = done ? reinterpret_cast<float*>(ring) : scratch0 + warp * (A.cols * D);
        if (done) {
          cp_wait<0>();
          __syncwarp();
        }
        if (lane == 0) {
          H.b = U.b;
          H.h = U.h;
          H.begins = run_begins;
          H.rest = U.rest;
          H.leads = warp == 0 && first_run;
          H.ncol = ncol;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int c = 0; c < CN; ++c) {
            const int col = col_of(n, c);
            if (col < ncol) {
              if (r == 0) {
                H.m[col] = m_run[n][c];
                H.l[col] = l_run[n][c];
              }
#pragma unroll
              for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int d = BITS == 16 ? 16 * i + 8 * h + r : 64 * (i / 4) + 8 * r + 2 * (i % 4) + h;
                  to[col * D + entry_at<BITS, HALF>(col, d)] = o_acc[n][i][2 * h + c];
                }
              }
            }
          }
        }
      }
      first_run = false;
    }
    st = st + 1 == STAGES ? 0 : st + 1;
  }

  // ---- join the warps' partial results, in the line's order. A warp takes a column: lane j holds entry j's
  // maximum and sum, the lanes of one (sequence, head) find their joint maximum together.
  cp_wait<0>();
  __syncthreads();
  const int my_b = lane < kWarps * 2 ? s_entry[lane].b : -1, my_h = lane < kWarps * 2 ? s_entry[lane].h : 0;
  const uint32_t valid = __ballot_sync(0xffffffffu, my_b >= 0);
  const uint32_t run = __match_any_sync(0xffffffffu, ((uint64_t)(uint32_t)my_b << 32) | (uint32_t)my_h) & valid;
  const uint32_t leaders = __ballot_sync(0xffffffffu, my_b >= 0 && (run & ((1u << lane) - 1)) == 0);
  for (int col = warp; col < A.cols; col += kWarps) {
    if (my_b >= 0) {
      const float mj = s_entry[lane].m[col], lj = s_entry[lane].l[col];
      int key = __float_as_int(mj);  // an order of integers that is the numbers' order
      key = key < 0 ? key ^ 0x7fffffff : key;
      key = __reduce_max_sync(run, key);
      const float joint = __int_as_float(key < 0 ? key ^ 0x7fffffff : key);
      const float f = weight_of(mj, lj, joint);
      s_f[lane][col] = f;
      s_fl[lane][col] = f * lj;
      s_entry[lane].m[col] = joint;
    }
  }
  __syncthreads();
  // The sums, 32 lanes times four values at a time, dealt over the warps in turn.
  int turn = warp;
  for (uint32_t later = leaders; later != 0; later &= later - 1) {
    const int n = __ffs(later) - 1;
    const uint32_t members = __shfl_sync(0xffffffffu, run, n);
    const EntryHead& H = s_entry[n];
    const int rest = s_entry[31 - __clz(members)].rest, ncol = H.ncol;
    const bool whole = H.begins && rest == 0;
    __nv_bfloat16* op = reinterpret_cast<__nv_bfloat16*>(A.out + (int64_t)H.b * A.out_stride) + (int64_t)H.h * D;
    // slot 0: the (sequence, head) that the CTA's run begins in; slot 1: another, which it ends in
    const int64_t slot = (int64_t)blockIdx.x * 2 + (H.leads ? 0 : 1);
    const int rounds = (ncol * (D / 4) + 31) / 32;
    const int first = turn;
    for (; turn < rounds; turn += kWarps) {
      const int i = turn * 32 + lane;  // four values of a column
      if (i >= ncol * (D / 4)) { continue; }
      const int col = i / (D / 4), d = (i % (D / 4)) * 4;
      const int at = col * (D / 4) + (entry_at<BITS, HALF>(col, d) >> 2);
      auto of = [&](int j) {
        return reinterpret_cast<const float4*>((j & 1) ? reinterpret_cast<const float*>(smem + (j >> 1) * A.ring_bytes)
                                                       : scratch0 + (j >> 1) * (A.cols * D))[at];
      };
      float l = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      auto add = [&](float f, float fl, const float4& x) {
        l += fl;
        acc.x = __fmaf_rn(f, x.x, acc.x), acc.y = __fmaf_rn(f, x.y, acc.y);
        acc.z = __fmaf_rn(f, x.z, acc.z), acc.w = __fmaf_rn(f, x.w, acc.w);
      };
      uint32_t k = members;
      for (; __popc(k) >= 4;) {  // four loads in flight
        int j[4];
        float4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          j[e] = __ffs(k) - 1;
          k &= k - 1;
          x[e] = of(j[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) { add(s_f[j[e]][col], s_fl[j[e]][col], x[e]); }
      }
      for (; k != 0; k &= k - 1) {
        const int j = __ffs(k) - 1;
        add(s_f[j][col], s_fl[j][col], of(j));
      }
      if (BITS == 8) {  // entry_at exchanges values within the four
        if (col & (HALF ? 1 : 2)) { acc = make_float4(acc.y, acc.x, acc.w, acc.z); }
        if (col & (HALF ? 2 : 4)) { acc = make_float4(acc.z, acc.w, acc.x, acc.y); }
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint2*>(op + i * 4) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4*>(A.part + slot * A.cols * D + i * 4) = acc;
        if (d == 0) {
          A.ml[(slot * A.cols + col) * 2] = H.m[col];
          A.ml[(slot * A.cols + col) * 2 + 1] = l;
        }
      }
    }
    turn -= rounds;
    if (!whole && H.begins && first == 0 && lane == 0) {
      A.heads[blockIdx.x] = {H.b, H.h, ncol * 2 + (H.leads ? 0 : 1), (int)div_u(cta1 + rest - 1, per_cta)};
    }
  }
}

// Joins what several CTAs have of a (sequence, head): block (c, col) serves column col of the one that
// begins in CTA c's run, its eight warps take every eighth part. Rows of sequences without a token get
// their zeros here, while the first kernel still runs.
constexpr int kJoinWarps = 8;
template <int D, int U>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attn_join_kernel(const AttnArgs A, int q_heads) {
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps], s_acc[kJoinWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x, col = blockIdx.y;
  if (col == 0) {
    // the first kernel has let this one start after what was before it had finished: lengths may be read
    for (int b = c0; b < A.batch; b += gridDim.x) {
      int s, n;
      token_range(A, b, s, n);
      if (n > s) { continue; }
      uint4* row = reinterpret_cast<uint4*>(A.out + (int64_t)b * A.out_stride);
      for (int i = threadIdx.x; i < q_heads * (D / 8); i += kJoinWarps * 32) { row[i] = make_uint4(0, 0, 0, 0); }
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // A warp's first part is fetched together with the record that says whether there is one (whatever lies
  // there is inside the workspace); the record's own CTA may have it in slot 1. The others four at a time.
  constexpr int V = D / 32;  // a lane's values: V neighbours
  struct Part {
    float m, l, x[V];
  };
  auto fetch = [&](Part& p, int64_t slot) {
    p.m = A.ml[slot * 2];
    p.l = A.ml[slot * 2 + 1];
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 w = *reinterpret_cast<const float2*>(A.part + slot * D + lane * V + i);
      p.x[i] = w.x, p.x[i + 1] = w.y;
    }
  };
  Part first;
  fetch(first, (int64_t)min(c0 + warp, (int)gridDim.x - 1) * 2 * A.cols + col);
  const CtaHead H = A.heads[c0];
  if (H.last < 0 || col >= (H.ncol_slot >> 1)) { return; }
  if (warp == 0 && (H.ncol_slot & 1)) { fetch(first, ((int64_t)c0 * 2 + 1) * A.cols + col); }
  float m = kNegInf, l = 0.0f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) { acc[i] = 0.0f; }
  auto add = [&](const Part& p) {
    const float m2 = fmaxf(m, p.m);
    const float f0 = weight_of(m, l, m2), f1 = weight_of(p.m, p.l, m2);
    m = m2;
    l = __fmaf_rn(f1, p.l, f0 * l);
#pragma unroll
    for (int i = 0; i < V; ++i) { acc[i] = __fmaf_rn(f1, p.x[i], f0 * acc[i]); }
  };
  if (c0 + warp <= H.last) { add(first); }
  for (int c = c0 + warp + kJoinWarps; c <= H.last; c += 4 * kJoinWarps) {
    Part p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) { fetch(p[k], (int64_t)min(c + k * kJoinWarps, H.last) * 2 * A.cols + col); }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (c + k * kJoinWarps <= H.last) { add(p[k]); }
    }
  }
  if (lane == 0) { s_m[warp] = m, s_l[warp] = l; }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { s_acc[warp][lane * V + i] = acc[i]; }
  __syncthreads();
  if (threadIdx.x >= D) { return; }
  float top = kNegInf, sum = 0.0f, o = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) { top = fmaxf(top, s_m[w]); }
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float f = weight_of(s_m[w], s_l[w], top);
    sum = __fmaf_rn(f, s_l[w], sum);
    o = __fmaf_rn(f, s_acc[w][threadIdx.x], o);
  }
  __nv_bfloat16* op = reinterpret_cast<__nv_bfloat16*>(A.out + (int64_t)H.b * A.out_stride) + (int64_t)(H.h + col) * D;
  op[threadIdx.x] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : o / sum);
}

// ---------------------------------------------------------------- host side
struct Shape {
  int group, cols, nt, blocks, ctas;
  int64_t capacity;  // tokens that a row of the page table can name
  size_t heads, ml, part, scratch, total;  // byte offsets in the workspace, and its size
};
constexpr int kMaxWarps = 16;  // of any instantiation: the scratch has room for them

int shape_of(const char* who, const vpq_paged_attention_desc* d, const vpq_kv_cache* c, Shape* s) {
  if (!d || !c) { return fail(VPQ_ERR_INVALID_ARG, "%s: null descriptor", who); }
  if (d->batch <= 0 || d->max_pages <= 0 || d->q_heads <= 0 || c->kv_heads <= 0 || d->q_heads % c->kv_heads) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: need batch>0, max_pages>0, q_heads a multiple of kv_heads (batch=%d max_pages=%d q_heads=%d kv_heads=%d)",
                who, d->batch, d->max_pages, d->q_heads, c->kv_heads);
  }
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256 (got %d)", who, c->head_dim);
  }
  if (d->q_heads > 65536) { return fail(VPQ_ERR_UNSUPPORTED, "%s: at most 65536 query heads", who); }
  s->group = d->q_heads / c->kv_heads;
  // Two column blocks of eight share a read of the cache where the accumulators leave room (head_dim
  // 256 has 64 of them per block). Wider groups read it again, from HBM where a sequence is long: 64 sequences of 4096 tokens,
  // four key heads, 16 bits, 8 / 16 query heads a key head at head_dim 256 1.08 / 2.15 GB and 172 / 329 us, 16 / 32 at
  // head_dim 128 0.54 / 1.08 GB and 97.5 / 178 us.
  s->nt = (s->group > 8 && c->head_dim <= 128) ? 2 : 1;
  s->cols = s->group < 8 * s->nt ? s->group : 8 * s->nt;
  s->blocks = (s->group + s->cols - 1) / s->cols;
  s->ctas = num_sms();
  s->capacity = (int64_t)d->max_pages * c->page_size;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t row = (size_t)s->cols * c->head_dim * 4;
  s->heads = 0;
  s->ml = up((size_t)s->ctas * sizeof(CtaHead));
  s->part = s->ml + up((size_t)s->ctas * 2 * s->cols * 8);
  s->scratch = s->part + up((size_t)s->ctas * 2 * row);
  s->total = s->scratch + up((size_t)s->ctas * kMaxWarps * row);
  return VPQ_OK;
}

template <int D, int BITS, int NT, bool HALF, int TM, int kWarps, int STAGES>
int launch(const AttnArgs& a0, const Shape& s, int q_heads, cudaStream_t st) {
  static_assert(kWarps <= kMaxWarps, "the workspace is sized for kMaxWarps");
  static_assert(NT * 8 * D * 4 <= STAGES * 2 * 16 * TM * (D * BITS / 8), "a warp's partial result fits its ring");
  constexpr int kStage = 2 * 16 * TM * (D * BITS / 8) + (BITS == 8 ? 2 * 16 * TM * (D / kKvGroup) * 4 : 0);
  constexpr int kRoom = 227 * 1024 - kWarps * 1216;  // beside what the kernel declares (at most 1136 bytes a warp)
  static_assert(kWarps * STAGES * (kStage + NT * 8 * D * 2) <= kRoom, "rings fit beside the static shared memory");
  AttnArgs a = a0;
  a.stage_bytes = kStage + ((s.cols * D * 2 + 127) & ~127);
  a.ring_bytes = a.stage_bytes * STAGES;
  static int granted[64] = {};
  auto kern = paged_attn_kernel<D, BITS, NT, HALF, TM, kWarps, STAGES>;
  size_t smem = (size_t)kWarps * a.ring_bytes;
  const size_t first = (size_t)kWarps * s.cols * D * 4;
  if (smem + first <= (size_t)kRoom) {
    smem += first;
    a.scratch = nullptr;
  }
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), granted, smem)) { return rc; }
  cudaLaunchConfig_t cfg = {};
  // Solo: a CTA has all of a (sequence, column block), so nothing spans CTAs and the second kernel and the line are saved
  // (3 us), but the machine is used as far as there are such CTAs and no longer than the longest lasts. Measured, solo against
  // the line, four query heads a key head unless said, a table as wide as the sequences:
  //   8 warps (128, bf16), 8 CTAs of 64 / 256 / 512 / 1024 tokens 3.7 / 5.3 / 6.9 / 10.0 us against 7.0 / 7.2 / 7.3 / 7.8, 128 CTAs
  //     3.9 / 5.5 / 7.2 / 10.5 against 7.5 / 9.1 / 10.7 / 13.9; (128, 8 bits), 8 CTAs of 512 / 1024 6.7 / 9.6 against 7.8 / 7.9;
  //     (256, 8 bits), 8 CTAs of 256 / 512 7.3 / 10.1 against 9.2 / 9.0, 128 CTAs of 512 / 1024 10.6 / 16.0 against 14.7 / 20.2;
  //   16 warps (64, bf16), 8 CTAs of 1024 / 2048 7.3 / 10.4 against 7.8 / 8.5, 128 CTAs 7.7 / 11.4 against 11.0 / 13.8; 8 bits alike;
  //   12 warps (64, 8 bits, 12 heads), 8 CTAs of 512 / 1024 7.5 / 10.5 against 10.1 / 10.0, 128 CTAs of 1024 11.1 against 15.2;
  //   5 warps (256, bf16), 8 CTAs of 256 / 512 7.9 / 11.2 against 8.5 / 8.7, 128 CTAs of 512 / 1024 11.7 / 24.6 against 15.7 / 29.8.
  // The lengths are the device's, so the rule goes by the longest that the table or the window allows, and stops at twice
  // what suits a few CTAs: one long sequence among short ones would hold the call up. (Of all these it takes the slower
  // side for 512 tokens of (256, 8 bits), by 1 us, and for 1024 of (256, bf16) in 128 CTAs.)
  const int64_t longest = a.window > 0 ? std::min<int64_t>((int64_t)a.window + 16 * TM, s.capacity) : s.capacity;
  const int64_t solo_ctas = (int64_t)a.batch * a.hk, suits = 64 * kWarps;
  a.solo = solo_ctas <= s.ctas && longest <= 2 * suits && longest * (s.ctas - solo_ctas) <= suits * s.ctas;
  cfg.gridDim = dim3((unsigned)(a.solo ? solo_ctas : s.ctas), 1, 1);
  cfg.blockDim = dim3(kWarps * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VPQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a));
  if (a.solo) { return VPQ_OK; }
  cfg.gridDim = dim3((unsigned)s.ctas, (unsigned)s.cols, 1);
  cfg.blockDim = dim3(kJoinWarps * 32, 1, 1);
  cfg.dynamicSmemBytes = 0;
  VPQ_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<D, 16 * TM>, a, q_heads));
  return VPQ_OK;
}

}  // namespace

}  // namespace vpq

using namespace vpq;

extern "C" size_t vpq_paged_attention_bytes(const vpq_paged_attention_desc* desc_host, const vpq_kv_cache* cache_host) {
  clear_error();
  Shape s = {};
  if (shape_of("paged_attention_bytes", desc_host, cache_host, &s) != VPQ_OK) { return 0; }
  clear_error();
  return s.total;
}

extern "C" int vpq_paged_attention_bf16(const vpq_paged_attention_desc* desc_host, const vpq_kv_cache* cache_host,
                                        void* workspace, size_t bytes, void* stream) {
  const char* who = "paged_attention";
  clear_error();
  Shape s = {};
  if (int rc = shape_of(who, desc_host, cache_host, &s)) { return rc; }
  const vpq_paged_attention_desc& d = *desc_host;
  AttnArgs a = {};
  if (int rc = kv_check(who, cache_host, &a.kv)) { return rc; }
  const int64_t row = (int64_t)d.q_heads * cache_host->head_dim;
  const int64_t qs = d.q_stride ? d.q_stride : row, os = d.out_stride ? d.out_stride : row;
  const int64_t ts = d.table_stride ? d.table_stride : d.max_pages;
  if (!d.q || !d.out || !d.page_table || !d.seq_lens || !workspace) { return fail(VPQ_ERR_INVALID_ARG, "%s: null pointer", who); }
  if (qs < row || os < row || ts < d.max_pages || qs > ((int64_t)1 << 46) / d.batch || os > ((int64_t)1 << 46) / d.batch ||
      ts > ((int64_t)1 << 46) / d.batch) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: a row stride is smaller than a row or out of range", who);
  }
  if (d.window < 0) { return fail(VPQ_ERR_INVALID_ARG, "%s: window must not be negative", who); }
  if ((int64_t)d.max_pages * cache_host->page_size > INT_MAX - 64) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: max_pages * page_size must stay below 2^31", who);
  }
  const float scale = d.scale != 0.0f ? d.scale : 1.0f / sqrtf((float)cache_host->head_dim);
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale >= FLT_MIN) || !(scale_log2 <= FLT_MAX)) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: scale must be 0 (1 / sqrt(head_dim)) or from 2^-126 to 2.3586e38 (got %g)", who, (double)d.scale);
  }
  if (!aligned16(d.q) || !aligned16(d.out) || (qs & 7) || (os & 7) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(d.page_table) & 3) || (reinterpret_cast<uintptr_t>(d.seq_lens) & 3)) {
    return fail(VPQ_ERR_ALIGNMENT, "%s: q, out, their row strides and the workspace must be multiples of 16 bytes", who);
  }
  if (bytes < s.total) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu are needed", who, bytes, s.total);
  }
  if (int rc = require_sm100()) { return rc; }
  if (int rc = index_status_word(&a.status)) { return rc; }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = static_cast<const uint8_t*>(d.q);
  a.out = static_cast<uint8_t*>(d.out);
  a.q_stride = qs * 2;
  a.out_stride = os * 2;
  a.page_table = d.page_table;
  a.seq_lens = d.seq_lens;
  a.table_stride = ts;
  a.heads = reinterpret_cast<CtaHead*>(ws + s.heads);
  a.ml = reinterpret_cast<float*>(ws + s.ml);
  a.part = reinterpret_cast<float*>(ws + s.part);
  a.scratch = reinterpret_cast<float*>(ws + s.scratch);
  a.batch = d.batch;
  a.max_pages = d.max_pages;
  a.window = d.window;
  a.group = s.group;
  a.cols = s.cols;
  a.blocks = s.blocks;
  a.hk = cache_host->kv_heads * s.blocks;
  a.dense = a.kv.token_bytes == (uint32_t)(cache_host->head_dim * cache_host->bits / 8) &&
            (cache_host->bits == 16 || a.kv.stoken_bytes == (uint32_t)(cache_host->head_dim / kKvGroup * 4));
  a.cta_rcp = (uint32_t)((((uint64_t)1 << 32) + s.ctas - 1) / s.ctas);
  a.few = d.batch <= 32 && (int64_t)d.max_pages * cache_host->page_size <= INT_MAX / 4;
  a.scale_log2 = scale_log2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool q8 = cache_host->bits == 8, two = s.nt == 2;
  const int qh = d.q_heads;
  // Tokens of a unit, warps and stages. A stage holds 8 to 16 KB, so that a warp's copies in flight cover the
  // latency; the warps' rings fill the shared memory. Measured at head_dim 128, warps x stages: 16 bits, 64 sequences of 1 to
  // 16384 tokens, 8 x 2 / 10 x 2 / 6 x 3 / 4 x 4 in 89.9 / 89.0 / 89.7 / 95.2 us, one of 333 tokens 5.7 / 6.1 / 6.2 / 6.8; 8 bits,
  // one of 131071 tokens, 8 x 2 / 10 x 2 / 6 x 3 in 52.0 / 54.8 / 58.9, and 58.2 with units of 16 tokens and 16 x 2. 64 sequences of
  // 4096 tokens, eight key heads with four query heads each (head_dim 256: four) unless said: head_dim 64, 16 bits, 16 x 2 / 12 x 2 /
  // 8 x 3 86.9 / 88.7 / 88.3; 8 bits, 16 x 2 / 12 x 2 / 8 x 2 54.0 / 55.0 / 64.3; twelve query heads, 16 bits, 8 x 3 / 8 x 2 / 12 x 2 /
  // 16 x 2 101 / 104.5 / 92.5 / 93.3, 8 bits, 12 x 2 / 8 x 2 / 16 x 2 82.6 / 88.0 / 109.4; head_dim 256, 16 bits, 5 x 2 / 4 x 2 / 3 x 2
  // 163.9 / 167.1 / 178.7, 8 bits, 8 x 2 / 6 x 2 / 5 x 3 95.3 / 110.7 / 129.4.
  const bool half = s.cols <= 4;
#define VPQ_GO(D, BITS, TM, W, S)                                    \
  if (half) { return launch<D, BITS, 1, true, TM, W, S>(a, s, qh, st); } \
  return launch<D, BITS, 1, false, TM, W, S>(a, s, qh, st);
  switch (cache_host->head_dim) {
    case 64:
      if (two) { return q8 ? launch<64, 8, 2, false, 2, 12, 2>(a, s, qh, st) : launch<64, 16, 2, false, 1, 8, 3>(a, s, qh, st); }
      if (q8) { VPQ_GO(64, 8, 2, 16, 2) }
      VPQ_GO(64, 16, 1, 16, 2)
    case 128:
      if (two) { return q8 ? launch<128, 8, 2, false, 2, 8, 2>(a, s, qh, st) : launch<128, 16, 2, false, 1, 8, 2>(a, s, qh, st); }
      if (q8) { VPQ_GO(128, 8, 2, 8, 2) }
      VPQ_GO(128, 16, 1, 8, 2)
    default:
      if (q8) { VPQ_GO(256, 8, 1, 8, 2) }
      VPQ_GO(256, 16, 1, 5, 2)
  }
#undef VPQ_GO
}
