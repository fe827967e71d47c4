// paged_attn.cu -- attention of one new token per sequence over a paged key-value cache.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,   p_t = 2^(log2(e) scale q_h . k_t - m),  m the running maximum
//
// Bound: HBM. Every key and value is read once and used by the q_heads / kv_heads queries that share
// it; per 16 tokens of one head that is 8 KB (bf16, head_dim 128) against 16 small matrix products.
//
// Work split. The unit is 16 tokens of one (sequence, key head). All units of a call, in the order
// (sequence, head, tokens), form one line that is cut into equal runs, one per CTA, and a CTA's run into one per
// warp: no SM waits for a long sequence, whatever the lengths, and the lengths are read on the device, so a
// captured graph serves any of them. Each warp streams its run through its own ring in shared memory
// (cp.async, no barrier in the loop). What a warp has of a (sequence, head) that it shares with others is
// joined within the CTA through shared memory, and across CTAs by a second small kernel over partial
// results in the workspace; both joins add in the line's order, so results do not depend on timing.
//
// Matrix products are m16n8k16 with the TOKENS as the 16 rows and up to eight query heads as the eight
// columns (a GQA group of four or eight wastes half or nothing; queries as rows would waste three quarters
// and need twice the accumulators). S^T = K Q^T comes out with tokens in rows; P enters the second product,
// O^T = V^T P^T, as its B operand, which wants the 8 x 8 blocks transposed: one movmatrix each.
//
// 8-bit caches multiply the codes, not the values: c - 128 is exact in fp16, so with k = s c + b
//   q . k = sum_g s_g (q . (c - 128))_g + (b_g + 128 s_g) sum_g q            (g: groups of 64)
//   o     = sum_t (p_t s_tg) (c - 128) + sum_t p_t (b_tg + 128 s_tg)
// and scales and biases act on 16 x 8 scores instead of 16 x head_dim values. Centred codes matter: with
// 0..255 the rounding of p s would be amplified by the codes' mean. q is scaled by a power of two per head to
// fill fp16's range (exact up to 2^-39 of the head's largest value); p s is taken relative to a running
// power of two above every scale, times 2^15, which keeps its rounding at 2^-11 relative down to 2^-29.
// In a bf16 cache p is rounded to bf16 (2^-8) and the sum of weights adds the rounded p, so the
// weights still sum to one.
#include "vpq_kv.cuh"
#include "vpq_sm100.cuh"

#include <climits>

namespace vpq {

__device__ uint32_t g_attn_status = 0;

namespace {

constexpr int kUnit = 16;    // tokens of a unit
constexpr float kNegInf = -__builtin_huge_valf();

struct AttnArgs {
  KvView kv;
  const uint8_t* q;
  uint8_t* out;
  int64_t q_stride, out_stride;  // bytes
  const int32_t* page_table;
  const int32_t* seq_lens;
  int64_t table_stride;
  int64_t* prefix;   // workspace: units (of one head) before each sequence, then units per CTA
  float* ml;         // [CTA][2][heads per column block][2]: maximum and sum of a partial result
  float* part;       // [CTA][2][heads per column block][D]
  int batch, max_pages, window;
  int group;         // query heads of a key head
  int cols;          // query heads a unit serves (a column block): min(group, 8 NT)
  int blocks;        // column blocks of a key head
  int hk;            // kv_heads * blocks
  float scale_log2;
  int stage_bytes, ring_bytes, entry_bytes;  // shared memory: a stage, a warp's ring, a partial result
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
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
// Bytes 0, 1 of w (HI: 2, 3) as fp16 pairs of c - 128: 0x6400 | c is 1024 + c exactly.
template <bool HI>
__device__ __forceinline__ uint32_t centred(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));  // 1152
  return r;
}

// Tokens of sequence b that count: [start, len), len cut to what the table can name.
__device__ __forceinline__ void token_range(const AttnArgs& A, int b, int& start, int& len) {
  int n = __ldg(A.seq_lens + b);
  const int64_t cap = (int64_t)A.max_pages * A.kv.page_size;
  if ((int64_t)n > cap) { n = (int)cap; }
  len = n > 0 ? n : 0;
  start = (A.window > 0 && len > A.window) ? len - A.window : 0;
}
__device__ __forceinline__ int units_of(int start, int len) { return len > start ? (len + kUnit - 1) / kUnit - start / kUnit : 0; }

// Where 16-byte chunk c of row `row` lies in a K or V tile. 16 bits: the eight rows that an ldmatrix
// reads fall into eight bank groups. 8 bits: see the loads in the loop.
template <int D, int BITS>
__device__ __forceinline__ int swz_k(int row, int c) {
  return BITS == 16 ? (c ^ (row & 7)) : (D >= 128 ? (c ^ ((row & 1) << 2)) : c);
}
template <int D, int BITS>
__device__ __forceinline__ int swz_v(int row, int c) {
  return BITS == 16 ? (c ^ (row & 7)) : (D >= 128 ? (c ^ (row & 6)) : (c ^ (row & 2)));
}

// What a unit in flight is: written by lane 0 with its copies, read when its turn comes.
struct alignas(16) UnitMeta {
  int b, h;       // sequence; key head * blocks + column block
  int lo_hi;      // live rows [lo, hi) of the 16
  int flags;
};
enum : int { kFirst = 1, kLast = 2, kSegBegin = 4, kSegEnd = 8 };

// A partial result of a warp, in shared memory: header here, D values of each column in the entry.
struct EntryHead {
  int seg;      // b * hk + h, -1: none
  int flags;    // kSegBegin, kSegEnd
  int b, h;
  float m[16], l[16];
};

template <int D, int BITS, int NT, int kWarps, int STAGES>
__global__ void __launch_bounds__(kWarps * 32, 1) paged_attn_kernel(const AttnArgs A) {
  constexpr int kRow = D * BITS / 8;
  constexpr int kTile = kUnit * kRow;
  constexpr int kPair = BITS == 8 ? D / kKvGroup * 4 : 0;  // scale pairs of a row
  constexpr int kPairs = kUnit * kPair;
  constexpr int G = D / kKvGroup;
  constexpr int MT = D / 16;  // 16-row blocks of O^T

  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_excl[kWarps * 32];
  __shared__ int64_t s_wsum[kWarps];
  __shared__ UnitMeta s_meta[kWarps][STAGES];
  __shared__ EntryHead s_entry[kWarps * 2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, t = lane & 3;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run of the line of units
  const int cpt = (A.batch + kWarps * 32 - 1) / (kWarps * 32);
  const int b_lo = min(tid * cpt, A.batch), b_hi = min(b_lo + cpt, A.batch);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    int s, n;
    token_range(A, b, s, n);
    mine += units_of(s, n);
  }
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) { incl += o; }
  }
  if (lane == 31) { s_wsum[warp] = incl; }
  if (tid < kWarps * 2) { s_entry[tid].seg = -1; }
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) { base += s_wsum[w]; }
    total += s_wsum[w];
  }
  const int64_t excl = base + incl - mine;
  s_excl[tid] = excl;
  const int64_t units = total * A.hk;
  int64_t per_cta = (units + gridDim.x - 1) / gridDim.x;
  per_cta = per_cta > kWarps ? per_cta : kWarps;
  if (blockIdx.x == 0) {  // what the joining kernel needs of this
    int64_t at = excl;
    for (int b = b_lo; b < b_hi; ++b) {
      int s, n;
      token_range(A, b, s, n);
      A.prefix[b] = at;
      at += units_of(s, n);
      if (__ldg(A.seq_lens + b) > n) { atomicOr(&g_attn_status, kBadLength); }
    }
    if (tid == 0) {
      A.prefix[A.batch] = total;
      A.prefix[A.batch + 1] = per_cta;
    }
  }
  __syncthreads();
  const int64_t cta0 = (int64_t)blockIdx.x * per_cta;
  if (cta0 >= units) { return; }  // the whole CTA
  const int64_t cta1 = cta0 + per_cta < units ? cta0 + per_cta : units;
  const int64_t per_warp = (cta1 - cta0 + kWarps - 1) / kWarps;
  const int64_t u0 = cta0 + warp * per_warp;
  int64_t u1 = u0 + per_warp < cta1 ? u0 + per_warp : cta1;
  int left = u0 < u1 ? (int)(u1 - u0) : 0;  // units this warp has yet to request
  int todo = left;                          // and to compute

  // ---- the loader's place in the line
  int lb = 0, lh = 0, ltile = 0, ltile0 = 0, ltile_end = 0, lstart = 0, llen = 0;
  int pg = 0, off = 0;     // page-table column and token offset in the page
  bool fresh = true;       // the next unit begins a (sequence, head) for this warp
  if (left > 0) {
    int lo = 0, hi = kWarps * 32 - 1;
    while (lo < hi) {  // the last thread whose sequences begin at or before u0
      const int mid = (lo + hi + 1) >> 1;
      if (s_excl[mid] * A.hk <= u0) {
        lo = mid;
      } else {
        hi = mid - 1;
      }
    }
    int64_t at = s_excl[lo];
    for (lb = lo * cpt;; ++lb) {
      token_range(A, lb, lstart, llen);
      const int n = units_of(lstart, llen);
      if ((at + n) * A.hk > u0) { break; }
      at += n;
    }
    ltile0 = lstart / kUnit;
    ltile_end = ltile0 + units_of(lstart, llen);
    const int64_t in_seq = u0 - at * A.hk;
    lh = (int)(in_seq / (ltile_end - ltile0));
    ltile = ltile0 + (int)(in_seq % (ltile_end - ltile0));
    pg = (int)((int64_t)ltile * kUnit / A.kv.page_size);
    off = (int)((int64_t)ltile * kUnit - (int64_t)pg * A.kv.page_size);
  }

  uint8_t* ring = smem + warp * A.ring_bytes;
  const uint32_t ring_s = smem_u32(ring);
  uint8_t* entry0 = smem + kWarps * A.ring_bytes + warp * A.entry_bytes;

  // Requests the next unit into stage `st`; commits a group in any case.
  auto request = [&](int st) {
    if (left > 0) {
      const int page = __ldg(A.page_table + (int64_t)lb * A.table_stride + pg);
      const bool ok = (uint32_t)page < (uint32_t)A.kv.num_pages;
      if (!ok && lane == 0) { atomicOr(&g_attn_status, kBadPage); }
      int lo = lstart - ltile * kUnit;
      lo = lo > 0 ? lo : 0;
      int hi = llen - ltile * kUnit;
      hi = hi < kUnit ? hi : kUnit;
      if (!ok) { lo = hi = 0; }
      const int64_t pp = ok ? page : 0;
      const int kvh = lh / A.blocks;
      const int64_t o = pp * A.kv.page_bytes + kvh * A.kv.head_bytes + (int64_t)off * A.kv.token_bytes;
      const uint32_t dst = ring_s + st * A.stage_bytes;
      constexpr int CH = kRow / 16;
#pragma unroll
      for (int j = 0; j < CH / 2; ++j) {
        const int id = lane + 32 * j, row = id / CH, c = id % CH;
        const bool live = row >= lo && row < hi;  // dead rows become zeros: whatever they hold, 0 p adds 0
        const int64_t so = o + row * A.kv.token_bytes + c * 16;
        cp_async16(dst + row * kRow + swz_k<D, BITS>(row, c) * 16, A.kv.k + so, live);
        cp_async16(dst + kTile + row * kRow + swz_v<D, BITS>(row, c) * 16, A.kv.v + so, live);
      }
      if (BITS == 8) {
        const int row = lane & 15;
        const bool live = row >= lo && row < hi;
        const uint8_t* sp = (lane < 16 ? A.kv.ks : A.kv.vs) + pp * A.kv.spage_bytes + kvh * A.kv.shead_bytes +
                            (int64_t)(off + row) * A.kv.stoken_bytes;
        cp_async_small<kPair ? kPair : 4>(dst + 2 * kTile + (lane < 16 ? 0 : kPairs) + row * kPair, sp, live);
      }
      if (fresh) {
        const int h0 = kvh * A.group + (lh % A.blocks) * A.cols;
        const int n = min(A.cols, A.group - (lh % A.blocks) * A.cols);
        const uint8_t* qp = A.q + (int64_t)lb * A.q_stride + (int64_t)h0 * (D * 2);
        for (int i = lane; i < n * (D / 8); i += 32) { cp_async16(dst + 2 * kTile + 2 * kPairs + i * 16, qp + i * 16, true); }
      }
      const bool last = left == 1 || ltile + 1 == ltile_end;
      if (lane == 0) {
        s_meta[warp][st] = {lb, lh, lo | (hi << 8),
                            (fresh ? kFirst : 0) | (last ? kLast : 0) | (ltile == ltile0 ? kSegBegin : 0) |
                                (ltile + 1 == ltile_end ? kSegEnd : 0)};
      }
      --left;
      fresh = false;
      off += kUnit;
      if (off == A.kv.page_size) { off = 0, ++pg; }
      if (++ltile == ltile_end && left > 0) {
        fresh = true;
        if (++lh == A.hk) {
          lh = 0;
          do {
            ++lb;
            token_range(A, lb, lstart, llen);
          } while (units_of(lstart, llen) == 0);
          ltile0 = lstart / kUnit;
          ltile_end = ltile0 + units_of(lstart, llen);
        }
        ltile = ltile0;
        pg = (int)((int64_t)ltile * kUnit / A.kv.page_size);
        off = (int)((int64_t)ltile * kUnit - (int64_t)pg * A.kv.page_size);
      }
    }
    cp_commit();
  };

  float o_acc[NT][MT][4];
  float m_run[NT][2], l_run[NT][2];
  float o_bias[NT][G][2], q_sum[NT][G][2], q_mul[NT][2];  // 8 bits
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
    const int ncol = min(A.cols, A.group - (U.h % A.blocks) * A.cols);

    if (U.flags & kFirst) {
      run_begins = (U.flags & kSegBegin) != 0;
      sigma = -100;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m_run[n][0] = m_run[n][1] = kNegInf;
        l_run[n][0] = l_run[n][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; ++i) { o_acc[n][i][0] = o_acc[n][i][1] = o_acc[n][i][2] = o_acc[n][i][3] = 0.0f; }
        const bool live = n * 8 + r < ncol;  // this lane's column
        const uint32_t qrow = qt + (n * 8 + r) * (D * 2);
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
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
#pragma unroll
            for (int i = 0; i < 2; ++i) { qf[n][k][i] = pack_f16x2(lo16(qf[n][k][i]) * up, hi16(qf[n][k][i]) * up); }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // the same for the columns of this lane's scores
            q_mul[n][c] = __shfl_sync(0xffffffffu, down, (2 * t + c) * 4);
#pragma unroll
            for (int g = 0; g < G; ++g) {
              q_sum[n][g][c] = __shfl_sync(0xffffffffu, sum[g], (2 * t + c) * 4);
              o_bias[n][g][c] = 0.0f;
            }
          }
        }
      }
    }

    // ---- scores: rows r, r + 8 of the unit, columns 2t, 2t + 1
    float s[NT][4];
    if (BITS == 16) {
#pragma unroll
      for (int n = 0; n < NT; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f; }
      const int row = (lane & 7) + (lane & 8), ch = lane >> 4;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t a[4];
        ldsm4(a, kt + row * kRow + swz_k<D, BITS>(row, 2 * k + ch) * 16);
#pragma unroll
        for (int n = 0; n < NT; ++n) { mma<false>(s[n], a, qf[n][k][0], qf[n][k][1]); }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { s[n][i] *= A.scale_log2; }
      }
    } else {
      float bias[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { s[n][i] = bias[n][i] = 0.0f; }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        // a lane's 16 codes feed four k steps: the k order is permuted the same way in q
        const uint4 x = lds128(kt + r * kRow + swz_k<D, BITS>(r, 4 * g + t) * 16);
        const uint4 y = lds128(kt + (r + 8) * kRow + swz_k<D, BITS>(r + 8, 4 * g + t) * 16);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
        float c[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) { c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f; }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t a[4] = {centred<false>(xs[u]), centred<false>(ys[u]), centred<true>(xs[u]), centred<true>(ys[u])};
#pragma unroll
          for (int n = 0; n < NT; ++n) { mma<true>(c[n], a, qf[n][g * 4 + u][0], qf[n][g * 4 + u][1]); }
        }
        const uint32_t p0 = lds32(ksc + r * kPair + g * 4), p1 = lds32(ksc + (r + 8) * kPair + g * 4);
        const float s0 = lo16(p0), s1 = lo16(p1);
        const float b0 = __fmaf_rn(128.0f, s0, hi16(p0)), b1 = __fmaf_rn(128.0f, s1, hi16(p1));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][i] = __fmaf_rn(c[n][i], i < 2 ? s0 : s1, s[n][i]);
            bias[n][i] = __fmaf_rn(i < 2 ? b0 : b1, q_sum[n][g][i & 1], bias[n][i]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { s[n][i] = __fmaf_rn(s[n][i], q_mul[n][i & 1], bias[n][i]) * A.scale_log2; }
      }
    }
    const int lo = U.lo_hi & 0xff, hi = U.lo_hi >> 8;
    const bool live0 = r >= lo && r < hi, live1 = r + 8 >= lo && r + 8 < hi;
    float p[NT][4];
    bool grows = false;
    float m_new[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) { s[n][i] = (i < 2 ? live0 : live1) ? s[n][i] : kNegInf; }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = fmaxf(s[n][c], s[n][2 + c]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        m_new[n][c] = fmaxf(m_run[n][c], x);
        grows |= m_new[n][c] > m_run[n][c];
      }
    }
    // 8 bits: this lane's value scales and centred biases
    float vs[2][G], vb[2][G], rescale = 1.0f, up = 1.0f;
    if (BITS == 8) {
      uint32_t top = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t p0 = lds32(vsc + r * kPair + g * 4), p1 = lds32(vsc + (r + 8) * kPair + g * 4);
        vs[0][g] = lo16(p0), vs[1][g] = lo16(p1);
        vb[0][g] = __fmaf_rn(128.0f, vs[0][g], hi16(p0));
        vb[1][g] = __fmaf_rn(128.0f, vs[1][g], hi16(p1));
        top = max(top, max((p0 << 16) & 0x7fffffffu, (p1 << 16) & 0x7fffffffu));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const int e = (int)(top >> 23) - 126;  // top < 2^e
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
        for (int c = 0; c < 2; ++c) {
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
      for (int i = 0; i < 4; ++i) {
        const float m = m_run[n][i & 1];
        p[n][i] = ex2(s[n][i] - (m == kNegInf ? 0.0f : m));  // no live token yet: 2^-inf, not NaN
      }
    }

    // ---- O^T += V^T P^T
    if (BITS == 16) {
      uint32_t b[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = pack_bf16x2(p[n][2 * h], p[n][2 * h + 1]);
          l_run[n][0] += lo16(w);
          l_run[n][1] += hi16(w);
          b[n][h] = movm(w);
        }
      }
      const int row = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t a[4];
        ldsm4t(a, vt + row * kRow + swz_v<D, BITS>(row, 2 * i + ch) * 16);
#pragma unroll
        for (int n = 0; n < NT; ++n) { mma<false>(o_acc[n][i], a, b[n][0], b[n][1]); }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { l_run[n][i & 1] += p[n][i]; }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t b[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = vs[h][g] * up;
            b[n][h] = movm(pack_f16x2(p[n][2 * h] * f, p[n][2 * h + 1] * f));
            o_bias[n][g][0] = __fmaf_rn(p[n][2 * h], vb[h][g], o_bias[n][g][0]);
            o_bias[n][g][1] = __fmaf_rn(p[n][2 * h + 1], vb[h][g], o_bias[n][g][1]);
          }
        }
        // codes 64 g + 8 r + 0..7 of tokens 2t, 2t + 1, 2t + 8, 2t + 9. A row's eight lanes of equal t read 64
        // bytes; the swizzle puts the four token pairs of a half warp into different banks.
        uint2 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 2 * t + (j & 1) + (j >> 1) * 8;
          w[j] = lds64(vt + row * kRow + swz_v<D, BITS>(row, 4 * g + (r >> 1)) * 16 + (r & 1) * 8);
        }
        uint32_t x[2][4];  // per token pair: values 0|1, 2|3, 4|5, 6|7 as bytes (even token, odd token, ...)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[h][0] = __byte_perm(w[2 * h].x, w[2 * h + 1].x, 0x5140);
          x[h][1] = __byte_perm(w[2 * h].x, w[2 * h + 1].x, 0x7362);
          x[h][2] = __byte_perm(w[2 * h].y, w[2 * h + 1].y, 0x5140);
          x[h][3] = __byte_perm(w[2 * h].y, w[2 * h + 1].y, 0x7362);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // rows r, r + 8 of this block: values 64 g + 8 r + 2 i, + 1
          const uint32_t a[4] = {centred<false>(x[0][i]), centred<true>(x[0][i]), centred<false>(x[1][i]),
                                 centred<true>(x[1][i])};
#pragma unroll
          for (int n = 0; n < NT; ++n) { mma<true>(o_acc[n][g * 4 + i], a, b[n][0], b[n][1]); }
        }
      }
    }

    // ---- the warp's part of a (sequence, head) is complete
    if (U.flags & kLast) {
      const bool run_ends = (U.flags & kSegEnd) != 0;
      const float o_mul = BITS == 8 ? __uint_as_float((uint32_t)(max(sigma - 15, -126) + 127) << 23) : 1.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
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
            for (int e = 0; e < 4; ++e) { o_acc[n][i][e] = __fmaf_rn(o_acc[n][i][e], o_mul, o_bias[n][i / 4][e & 1]); }
          }
        }
      }
      if (run_begins && run_ends) {
        const int h0 = (U.h / A.blocks) * A.group + (U.h % A.blocks) * A.cols;
        uint8_t* op = A.out + (int64_t)U.b * A.out_stride + (int64_t)h0 * (D * 2);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // a sum of 0: no live token (a NaN stays one)
          const float i0 = l_run[n][0] == 0.0f ? 0.0f : 1.0f / l_run[n][0];
          const float i1 = l_run[n][1] == 0.0f ? 0.0f : 1.0f / l_run[n][1];
          if (BITS == 16) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w = movm(pack_bf16x2(o_acc[n][i][2 * h] * i0, o_acc[n][i][2 * h + 1] * i1));
                if (n * 8 + r < ncol) {
                  *reinterpret_cast<uint32_t*>(op + (n * 8 + r) * (D * 2) + (16 * i + 8 * h + 2 * t) * 2) = w;
                }
              }
            }
          } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const float inv = c ? i1 : i0;
                const int col = n * 8 + 2 * t + c;
                uint4 y;
                y.x = pack_bf16x2(o_acc[n][g * 4][c] * inv, o_acc[n][g * 4][2 + c] * inv);
                y.y = pack_bf16x2(o_acc[n][g * 4 + 1][c] * inv, o_acc[n][g * 4 + 1][2 + c] * inv);
                y.z = pack_bf16x2(o_acc[n][g * 4 + 2][c] * inv, o_acc[n][g * 4 + 2][2 + c] * inv);
                y.w = pack_bf16x2(o_acc[n][g * 4 + 3][c] * inv, o_acc[n][g * 4 + 3][2 + c] * inv);
                if (col < ncol) { *reinterpret_cast<uint4*>(op + col * (D * 2) + (64 * g + 8 * r) * 2) = y; }
              }
            }
          }
        }
      } else {
        // at most two per warp: the first part of its run, kept apart, and the last, over the ring that
        // nothing is in flight to any more
        const int e = first_run ? 0 : 1;
        float* to = reinterpret_cast<float*>(first_run ? entry0 : ring);
        if (!first_run) {
          cp_wait<0>();
          __syncwarp();
        }
        EntryHead& H = s_entry[warp * 2 + e];
        if (lane == 0) {
          H.seg = U.b * A.hk + U.h;
          H.flags = (run_begins ? kSegBegin : 0) | (run_ends ? kSegEnd : 0);
          H.b = U.b;
          H.h = U.h;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int col = n * 8 + 2 * t + c;
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
                  to[col * D + d] = o_acc[n][i][2 * h + c];
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

  // ---- join the warps' partial results, in the line's order
  cp_wait<0>();
  __syncthreads();
  for (int item = warp; item < kWarps * 2 * A.cols; item += kWarps) {
    const int n = item / A.cols, col = item % A.cols;
    const EntryHead& H = s_entry[n];
    if (H.seg < 0 || col >= min(A.cols, A.group - (H.h % A.blocks) * A.cols)) { continue; }
    int prev = n - 1;
    while (prev >= 0 && s_entry[prev].seg < 0) { --prev; }
    if (prev >= 0 && s_entry[prev].seg == H.seg) { continue; }  // another item joins it
    int end = n, flags = 0;
    float m = kNegInf;
    for (int j = n; j < kWarps * 2; ++j) {
      if (s_entry[j].seg < 0) { continue; }
      if (s_entry[j].seg != H.seg) { break; }
      end = j;
      flags = s_entry[j].flags;
      m = fmaxf(m, s_entry[j].m[col]);
    }
    const bool whole = (H.flags & kSegBegin) && (flags & kSegEnd);
    float l = 0.0f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) { acc[i] = 0.0f; }
    for (int j = n; j <= end; ++j) {
      if (s_entry[j].seg < 0) { continue; }
      const float mj = s_entry[j].m[col];
      const float f = mj == kNegInf ? (s_entry[j].l[col] == 0.0f ? 0.0f : 1.0f) : ex2(mj - m);
      l = __fmaf_rn(f, s_entry[j].l[col], l);
      const float* from = reinterpret_cast<const float*>((j & 1) ? smem + (j >> 1) * A.ring_bytes
                                                                 : smem + kWarps * A.ring_bytes + (j >> 1) * A.entry_bytes);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) { acc[i] = __fmaf_rn(f, from[col * D + i * 32 + lane], acc[i]); }
    }
    if (whole) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int head = (H.h / A.blocks) * A.group + (H.h % A.blocks) * A.cols + col;
      __nv_bfloat16* op = reinterpret_cast<__nv_bfloat16*>(A.out + (int64_t)H.b * A.out_stride) + (int64_t)head * D;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) { op[i * 32 + lane] = __float2bfloat16_rn(acc[i] * inv); }
    } else {
      // slot 0: the (sequence, head) that the CTA's run begins in; slot 1: the one it ends in
      const int64_t slot = (int64_t)blockIdx.x * 2 + (n == 0 ? 0 : 1);
      float* pp = A.part + (slot * A.cols + col) * D;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) { pp[i * 32 + lane] = acc[i]; }
      if (lane == 0) {
        A.ml[(slot * A.cols + col) * 2] = m;
        A.ml[(slot * A.cols + col) * 2 + 1] = l;
      }
    }
  }
}

// Joins what several CTAs have of a (sequence, head): one warp per query head. Sequences without a
// token get their zeros here.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const AttnArgs A, int q_heads) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int b = (int)(id / q_heads), head = (int)(id % q_heads);
  if (b >= A.batch) { return; }
  const int kvh = head / A.group, blk = (head % A.group) / A.cols, col = (head % A.group) % A.cols;
  const int64_t p0 = A.prefix[b], n = A.prefix[b + 1] - p0, per_cta = A.prefix[A.batch + 1];
  __nv_bfloat16* op = reinterpret_cast<__nv_bfloat16*>(A.out + (int64_t)b * A.out_stride) + (int64_t)head * D;
  float acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { acc[i] = 0.0f; }
  float l = 0.0f;
  if (n > 0) {
    const int64_t u0 = p0 * A.hk + (kvh * A.blocks + blk) * n, u1 = u0 + n;
    const int64_t c0 = u0 / per_cta, c1 = (u1 - 1) / per_cta;
    if (c0 == c1) { return; }  // one CTA had it all and has written it
    auto slot_of = [&](int64_t c) { return (c * 2 + (c * per_cta < u0 ? 1 : 0)) * A.cols + col; };
    float m = kNegInf;
    for (int64_t c = c0 + lane; c <= c1; c += 32) { m = fmaxf(m, A.ml[slot_of(c) * 2]); }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) { m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d)); }
#pragma unroll 4
    for (int64_t c = c0; c <= c1; ++c) {
      const int64_t sl = slot_of(c);
      const float mj = A.ml[sl * 2], lj = A.ml[sl * 2 + 1];
      const float f = mj == kNegInf ? (lj == 0.0f ? 0.0f : 1.0f) : ex2(mj - m);
      l = __fmaf_rn(f, lj, l);
      const float* pp = A.part + sl * D;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) { acc[i] = __fmaf_rn(f, pp[i * 32 + lane], acc[i]); }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { op[i * 32 + lane] = __float2bfloat16_rn(acc[i] * inv); }
}

// ---------------------------------------------------------------- host side
struct Shape {
  int group, cols, nt, blocks, ctas;
  size_t prefix, ml, part, total;  // byte offsets in the workspace, and its size
};

int shape_of(const char* who, const vpq_paged_attention_desc* d, const vpq_kv_cache* c, Shape* s) {
  if (!d || !c) { return fail(VPQ_ERR_INVALID_ARG, "%s: null descriptor", who); }
  if (d->batch <= 0 || d->max_pages <= 0 || d->q_heads <= 0 || c->kv_heads <= 0 || d->q_heads % c->kv_heads) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: need batch>0, max_pages>0, q_heads a multiple of kv_heads (batch=%d max_pages=%d q_heads=%d kv_heads=%d)",
                who, d->batch, d->max_pages, d->q_heads, c->kv_heads);
  }
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256 (got %d)", who, c->head_dim);
  }
  if (d->q_heads > 65536 || (int64_t)d->batch * d->q_heads > INT_MAX / 2) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: at most 65536 query heads and 2^30 of them in a batch", who);
  }
  s->group = d->q_heads / c->kv_heads;
  // Two column blocks of eight share a read of the cache where the accumulators leave room (head_dim
  // 256 has 64 of them per block); wider groups read it again, from L2 for the most part.
  s->nt = (s->group > 8 && c->head_dim <= 128) ? 2 : 1;
  s->cols = s->group < 8 * s->nt ? s->group : 8 * s->nt;
  s->blocks = (s->group + s->cols - 1) / s->cols;
  s->ctas = num_sms();
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  s->prefix = 0;
  s->ml = up((size_t)(d->batch + 2) * 8);
  s->part = s->ml + up((size_t)s->ctas * 2 * s->cols * 8);
  s->total = s->part + up((size_t)s->ctas * 2 * s->cols * c->head_dim * 4);
  return VPQ_OK;
}

template <int D, int BITS, int NT, int kWarps, int STAGES>
int launch_main(const AttnArgs& a0, const Shape& s, cudaStream_t st) {
  AttnArgs a = a0;
  constexpr int kRow = D * BITS / 8;
  constexpr int kPairs = BITS == 8 ? kUnit * (D / kKvGroup) * 4 : 0;
  a.stage_bytes = 2 * kUnit * kRow + 2 * kPairs + ((s.cols * D * 2 + 127) & ~127);
  a.entry_bytes = s.cols * D * 4;
  a.ring_bytes = a.stage_bytes * STAGES;
  if (a.ring_bytes < a.entry_bytes) { a.ring_bytes = a.entry_bytes; }
  a.ring_bytes = (a.ring_bytes + 127) & ~127;
  const size_t smem = (size_t)kWarps * (a.ring_bytes + a.entry_bytes);
  static int granted[64] = {};
  auto kern = paged_attn_kernel<D, BITS, NT, kWarps, STAGES>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), granted, smem)) { return rc; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)s.ctas, 1, 1);
  cfg.blockDim = dim3(kWarps * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VPQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a));
  return VPQ_OK;
}

template <int D>
int launch_join(const AttnArgs& a, int q_heads, cudaStream_t st) {
  const int64_t warps = (int64_t)a.batch * q_heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((warps + 7) / 8), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VPQ_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<D>, a, q_heads));
  return VPQ_OK;
}

}  // namespace

int attn_status_read(cudaStream_t st, uint32_t* out) {
  uint32_t v = 0;
  VPQ_CUDA_OK(cudaMemcpyFromSymbolAsync(&v, g_attn_status, sizeof(v), 0, cudaMemcpyDeviceToHost, st));
  VPQ_CUDA_OK(cudaStreamSynchronize(st));
  if (v != 0) {
    const uint32_t zero = 0;
    VPQ_CUDA_OK(cudaMemcpyToSymbolAsync(g_attn_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st));
    VPQ_CUDA_OK(cudaStreamSynchronize(st));
  }
  *out = v;
  return VPQ_OK;
}

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
  if ((int64_t)d.max_pages * cache_host->page_size > INT_MAX - kUnit) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: max_pages * page_size must stay below 2^31", who);
  }
  if (!(d.scale >= 0.0f) || d.scale > 3.4e38f) { return fail(VPQ_ERR_INVALID_ARG, "%s: scale must be finite and not negative", who); }
  if (!aligned16(d.q) || !aligned16(d.out) || (qs & 7) || (os & 7) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(d.page_table) & 3) || (reinterpret_cast<uintptr_t>(d.seq_lens) & 3)) {
    return fail(VPQ_ERR_ALIGNMENT, "%s: q, out, their row strides and the workspace must be multiples of 16 bytes", who);
  }
  if (bytes < s.total) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu are needed", who, bytes, s.total);
  }
  if (int rc = require_sm100()) { return rc; }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = static_cast<const uint8_t*>(d.q);
  a.out = static_cast<uint8_t*>(d.out);
  a.q_stride = qs * 2;
  a.out_stride = os * 2;
  a.page_table = d.page_table;
  a.seq_lens = d.seq_lens;
  a.table_stride = ts;
  a.prefix = reinterpret_cast<int64_t*>(ws + s.prefix);
  a.ml = reinterpret_cast<float*>(ws + s.ml);
  a.part = reinterpret_cast<float*>(ws + s.part);
  a.batch = d.batch;
  a.max_pages = d.max_pages;
  a.window = d.window;
  a.group = s.group;
  a.cols = s.cols;
  a.blocks = s.blocks;
  a.hk = cache_host->kv_heads * s.blocks;
  const float scale = d.scale != 0.0f ? d.scale : 1.0f / sqrtf((float)cache_host->head_dim);
  a.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool q8 = cache_host->bits == 8, two = s.nt == 2;
  int rc = VPQ_OK;
  // Warps and stages by what fits 227 KB: eight warps, or four where a stage or the partial results are large.
  switch (cache_host->head_dim) {
    case 64:
      rc = q8 ? (two ? launch_main<64, 8, 2, 8, 4>(a, s, st) : launch_main<64, 8, 1, 8, 4>(a, s, st))
              : (two ? launch_main<64, 16, 2, 8, 3>(a, s, st) : launch_main<64, 16, 1, 8, 4>(a, s, st));
      if (rc == VPQ_OK) { rc = launch_join<64>(a, d.q_heads, st); }
      break;
    case 128:
      rc = q8 ? (two ? launch_main<128, 8, 2, 8, 2>(a, s, st) : launch_main<128, 8, 1, 8, 3>(a, s, st))
              : (two ? launch_main<128, 16, 2, 4, 3>(a, s, st) : launch_main<128, 16, 1, 8, 2>(a, s, st));
      if (rc == VPQ_OK) { rc = launch_join<128>(a, d.q_heads, st); }
      break;
    default:
      rc = q8 ? launch_main<256, 8, 1, 4, 3>(a, s, st) : launch_main<256, 16, 1, 4, 2>(a, s, st);
      if (rc == VPQ_OK) { rc = launch_join<256>(a, d.q_heads, st); }
      break;
  }
  return rc;
}
