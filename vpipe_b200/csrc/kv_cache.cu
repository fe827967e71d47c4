// kv_cache.cu -- norm of queries and keys per head with the position rotation, and the paged
// key-value cache's store (plain, or 8-bit affine) and load. All memory streams: a few dozen
// instructions per 16 bytes, each row read once and written once.
#include "vpq_kv.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace vpq {

namespace {

// How rows are dealt: a block belongs to one part (q, k or v; so what goes by the part is the same for all its
// threads), whose heads are cut into chunks of HPT neighbours; a lane group takes one chunk of every `step`-th
// token. A block holds the chunks of `tokens` whole tokens, or one token's chunks are spread evenly over
// `token_blocks` blocks.
struct Deal {
  uint32_t first;    // the part's first block
  int chunks;        // of a token
  int per_block;     // of a token in a block
  int tokens, token_blocks;
  uint32_t rcp;      // 2^16 / per_block, rounded up: (g * rcp) >> 16 = g / per_block for g < 256
  uint32_t step;     // tokens that the part's blocks take at a time
};
// The calling lane group's chunk, its first token and its block's; false if there is no chunk for it (such lanes
// keep their warp's shuffles company).
template <int LPH>
__device__ __forceinline__ bool dealt(const Deal& d, uint32_t& m0, uint32_t& tl, int& chunk) {
  const uint32_t g = threadIdx.x / LPH, blk = blockIdx.x - d.first;
  tl = (g * d.rcp) >> 16;
  const uint32_t tb = d.token_blocks == 1 ? blk : blk / (uint32_t)d.token_blocks;
  m0 = tb * (uint32_t)d.tokens;
  chunk = (int)((blk - tb * (uint32_t)d.token_blocks) * (uint32_t)d.per_block + (g - tl * d.per_block));
  const bool in = tl < (uint32_t)d.tokens && chunk < d.chunks;
  if (!in) { tl = 0, chunk = 0; }
  return in;
}
// p + a b, one instruction.
__device__ __forceinline__ uint8_t* at(const uint8_t* p, uint32_t a, uint32_t b) {
  return const_cast<uint8_t*>(p) + (uint64_t)a * b;
}

// One head's row is D values, eight (16 bytes) per lane: LPH = D / 8 lanes hold it, and every
// reduction (the norm's sum, a group's extremes) and the exchange of rotation partners is a shuffle
// among them. A head is processed in registers from load to store, so q_out = q is safe.
struct QkArgs {
  const uint8_t* in[3];  // q, k, v rows; null where there are none
  uint8_t* out[2];       // q, k rows out
  uint32_t in_stride[3];  // bytes
  uint32_t out_stride[2];
  const uint16_t* norm_w[2];
  const float* cos_sin;
  const int32_t* positions;
  const int64_t* slots;
  uint32_t M, table_rows;
  int64_t num_slots;
  int heads[3];
  Deal deal[3];
  int rot, interleaved;
  float eps, inv_d;
  KvView kv;
  uint32_t* status;  // index reports
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void unpack8(const uint4 r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// The 8-bit quantizer over the 64 values of eight lanes, from their extremes. The bias is the minimum rounded
// DOWN to bf16 and the scale is rounded UP, so min and max both lie inside the code range: with nearest rounding a
// group whose offset is large against its spread would lose values to clipping (the bias alone is off by up to 2^-8
// of the offset). The scale's floor of 2^-126 keeps its reciprocal finite; a group of equal values takes code 0. A
// NaN or infinity among the 64 (or a spread beyond the largest float) makes the pair NaN, so the group reads back as
// NaN. Directed rounding to bf16 is integer arithmetic on the bits; the quotient by 255 is rounded up exactly: a
// product with a factor a little above 1 / 255 is cut to bf16, and the next number up is taken if 255 times that
// (exact: 8 bits times 8) falls short.
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float mn, float mx, uint32_t& pair) {
  const uint32_t mb = __float_as_uint(mn);
  const uint32_t bb = (mb + ((uint32_t)((int32_t)mb >> 31) & 0xffffu)) & 0xffff0000u;
  const float b = __uint_as_float(bb);
  const float range = __fsub_rn(mx, b);
  const float cut = __uint_as_float(__float_as_uint(__fmul_rn(range, 0.0039215696f)) & 0xffff0000u);  // (1 + 2^-22) / 255
  const uint32_t up = __fmul_rn(cut, 255.0f) >= range ? 0u : 0x10000u;
  const float s = fmaxf(__uint_as_float(__float_as_uint(cut) + up), 1.17549435e-38f);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));  // within one step; s and 1 / s are normal numbers
  pair = range <= 3.402823466e38f ? (__float_as_uint(s) >> 16) | bb : 0x7fff7fffu;  // false for NaN
  // Adding 2^23 rounds to an integer, ties to even, and leaves it in the low byte: b <= x and the rounded-up
  // scale keep the quotient in [0, 255.0002], so there is nothing to clamp.
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x[i], b), inv), 8388608.0f)); }
  auto four = [](uint32_t a, uint32_t b2, uint32_t c2, uint32_t d) {
    return __byte_perm(__byte_perm(a, b2, 0x0040), __byte_perm(c2, d, 0x0040), 0x5410);
  };
  return make_uint2(four(c[0], c[1], c[2], c[3]), four(c[4], c[5], c[6], c[7]));
}
// The extremes of f32 values.
__device__ __forceinline__ uint2 quant8(const float (&x)[8], uint32_t& pair) {
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    mn = min_nan(mn, x[i]);
    mx = max_nan(mx, x[i]);
  }
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) {
    mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, d));
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  }
  return quant8(x, mn, mx, pair);
}
// Values that are bf16 already: extremes two at a time, then (minimum, -maximum) as one word.
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint2 quant8(const uint4 raw, uint32_t& pair) {
  constexpr uint32_t kSign = 0x80008000u;
  const uint32_t lo = min_nan2(min_nan2(raw.x, raw.y), min_nan2(raw.z, raw.w));
  const uint32_t hi = min_nan2(min_nan2(raw.x ^ kSign, raw.y ^ kSign), min_nan2(raw.z ^ kSign, raw.w ^ kSign));
  uint32_t m = min_nan2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) { m = min_nan2(m, __shfl_xor_sync(0xffffffffu, m, d)); }
  float x[8];
  unpack8(raw, x);
  return quant8(x, __uint_as_float(m << 16), -__uint_as_float(m & 0xffff0000u), pair);
}

// A slot inside the cache as page and place. (Pages and places fit 32 bits; a 64-bit division costs five times as much.)
__device__ __forceinline__ void split_slot(int64_t slot, const KvView& kv, uint32_t& page, uint32_t& place) {
  if (kv.page_shift >= 0) {
    page = (uint32_t)(slot >> kv.page_shift);
  } else {
    page = (slot >> 32) == 0 ? (uint32_t)slot / (uint32_t)kv.page_size : (uint32_t)(slot / kv.page_size);
  }
  place = (uint32_t)slot - page * (uint32_t)kv.page_size;
}

// MODE 0: q and k rows out. 16 / 8: q rows out, k and v into a cache of that width. HPT: heads of a chunk, all
// requested before the first is used; their table row, norm weights and addresses are fetched once.
// Bound by memory where rows go out as bf16: 16320 tokens of 40 + 40 heads of 128 in 106.7 us, 6.34 TB/s or 97 % of a
// copy's rate. Into an 8-bit cache the quantizer's instructions bound it: 8191 tokens of 32 + 8 + 8 heads of 128 in
// 39.4 us, 74 %. One token: 1.8 us (2.3 us with an 8-bit store), a launch and one chain of loads.
template <int D, int MODE, int HPT>
__global__ void __launch_bounds__(256, HPT > 1 ? 4 : 3) norm_rope_store_kernel(const __grid_constant__ QkArgs A) {
  constexpr int LPH = D / 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int part = MODE && blockIdx.x >= A.deal[2].first ? 2 : (blockIdx.x >= A.deal[1].first ? 1 : 0);
  const Deal& deal = A.deal[part];
  const int l = threadIdx.x % LPH, d0 = l * 8;
  uint32_t m0, tl;
  int chunk;
  const bool mine = dealt<LPH>(deal, m0, tl, chunk);
  const int h0 = HPT * chunk;
  const int n = min(HPT, A.heads[part] - h0);  // heads of this chunk
  const bool to_cache = MODE != 0 && part > 0;

  // This lane's eight values among the pairs: y = r (x cw + o sw), o the partner's values (in lane `partner`, or
  // the neighbours). The norm weights are folded into cos and sin, so that a head costs one product and one sum a
  // value, and the exchange does not wait for the norm.
  const int half = A.rot >> 1;
  const bool turns = A.cos_sin && part < 2, rotated = turns && d0 < A.rot;
  const bool swap = turns && !A.interleaved;
  const bool second = d0 >= half;
  const int partner = swap && rotated ? (second ? l - (half >> 3) : l + (half >> 3)) : l;
  const uint16_t* nw = part < 2 ? A.norm_w[part] : nullptr;
  uint32_t m = m0 + tl;
  // the longest chain first, and a token ahead: position, table row
  const bool by_position = A.cos_sin && A.positions;
  int p = 0;
  if (by_position && m < A.M) { p = __ldg(A.positions + m); }
  for (; m0 < A.M; m0 += deal.step, m += deal.step) {
    const bool live = mine && m < A.M;
    const uint32_t mm = live ? m : 0;  // a row to read in any case
    const uint8_t* in = at(A.in[part], mm, A.in_stride[part]) + (h0 * (D * 2) + l * 16);
    uint4 raw[HPT];
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      if (i > 0) { raw[i] = make_uint4(0, 0, 0, 0); }
      if (i == 0 || i < n) { raw[i] = *reinterpret_cast<const uint4*>(in + i * (D * 2)); }
    }
    bool turn = live;  // whether this token is written at all
    uint32_t row = mm;
    if (by_position) {
      turn = live && p >= 0 && (uint32_t)p < A.table_rows;
      if (live && p >= 0 && !turn && l == 0) { atomicOr(A.status, kBadPosition); }
      row = turn ? (uint32_t)p : 0;
      if (m + deal.step < A.M) { p = __ldg(A.positions + m + deal.step); }
    }
    float cw[8], sw[8];
    if (nw) {
      unpack8(__ldg(reinterpret_cast<const uint4*>(nw) + l), cw);
      unpack8(__ldg(reinterpret_cast<const uint4*>(nw) + partner), sw);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) { cw[e] = sw[e] = 1.0f; }
    }
    if (rotated) {
      const float* tab = reinterpret_cast<const float*>(at(reinterpret_cast<const uint8_t*>(A.cos_sin), row, A.rot * 4)) + (A.interleaved ? d0 >> 1 : (second ? d0 - half : d0));
      if (swap) {
        const float sg = second ? 1.0f : -1.0f;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 c = __ldg(reinterpret_cast<const float4*>(tab + e)), s = __ldg(reinterpret_cast<const float4*>(tab + half + e));
          cw[e] *= c.x, cw[e + 1] *= c.y, cw[e + 2] *= c.z, cw[e + 3] *= c.w;
          sw[e] *= sg * s.x, sw[e + 1] *= sg * s.y, sw[e + 2] *= sg * s.z, sw[e + 3] *= sg * s.w;
        }
      } else {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(tab)), s4 = __ldg(reinterpret_cast<const float4*>(tab + half));
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float wa = cw[2 * e], wb = cw[2 * e + 1];
          cw[2 * e] = wa * c[e], sw[2 * e] = -wb * s[e];
          cw[2 * e + 1] = wb * c[e], sw[2 * e + 1] = wa * s[e];
        }
      }
    }
    uint8_t* out;
    uint8_t* pairs = nullptr;
    if (to_cache) {
      const int64_t s = __ldg(A.slots + mm);
      if (live && s >= A.num_slots && l == 0) { atomicOr(A.status, kBadSlot); }
      turn = turn && s >= 0 && s < A.num_slots;
      uint32_t page = 0, place = 0;
      if (turn) { split_slot(s, A.kv, page, place); }
      out = at(at((part == 1 ? A.kv.k : A.kv.v) + page * A.kv.page_bytes, place, A.kv.token_bytes), h0, A.kv.head_bytes) +
            l * (MODE == 8 ? 8 : 16);
      if (MODE == 8) {
        pairs = at(at((part == 1 ? A.kv.ks : A.kv.vs) + page * A.kv.spage_bytes, place, A.kv.stoken_bytes), h0,
                   A.kv.shead_bytes) + (l >> 3) * 4;
      }
    } else {
      out = at(A.out[MODE ? 0 : part], mm, A.out_stride[MODE ? 0 : part]) + (h0 * (D * 2) + l * 16);
    }
    const uint32_t to_step = to_cache ? A.kv.head_bytes : D * 2;  // from a head to the next
    const int writes = turn ? n : 0;
    auto put_codes = [&](int i, uint2 c, uint32_t pair) {
      if (i < writes) {
        *reinterpret_cast<uint2*>(out + i * to_step) = c;
        if ((l & 7) == 0) { *reinterpret_cast<uint32_t*>(pairs + i * A.kv.shead_bytes) = pair; }
      }
    };
    if (MODE && part == 2) {  // values: as they are
#pragma unroll
      for (int i = 0; i < HPT; ++i) {
        if (MODE == 16) {
          if (i < writes) { *reinterpret_cast<uint4*>(out + i * to_step) = raw[i]; }
        } else {
          uint32_t pair;
          const uint2 c = quant8(raw[i], pair);
          put_codes(i, c, pair);
        }
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      float x[8], o[8];
      unpack8(raw[i], x);
      float r = 1.0f;
      if (nw) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) { ss = __fmaf_rn(x[e], x[e], ss); }
#pragma unroll
        for (int d = 1; d < LPH; d <<= 1) { ss += __shfl_xor_sync(0xffffffffu, ss, d); }
        r = rsqrtf(__fmaf_rn(ss, A.inv_d, A.eps));
      }
      if (swap) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { o[e] = __shfl_sync(0xffffffffu, x[e], partner, LPH); }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) { o[e] = x[e ^ 1]; }
      }
      if (rotated) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = __fmaf_rn(o[e], sw[e], x[e] * cw[e]) * r; }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = x[e] * cw[e] * r; }
      }
      if (MODE == 8 && to_cache) {
        uint32_t pair;
        const uint2 c = quant8(x, pair);
        put_codes(i, c, pair);
      } else if (i < writes) {
        *reinterpret_cast<uint4*>(out + i * to_step) = pack8(x);
      }
    }
  }
}

struct CopyArgs {
  KvView kv;
  uint8_t* rows[2];   // k, v: read by the store, written by the load
  uint32_t stride[2];  // bytes
  uint32_t M;
  const int64_t* slots;
  int64_t num_slots;
  uint32_t* status;  // index reports
  Deal deal[2];
};

// Rows into the cache (STORE), or out of it: eight values a lane and head, 8 bytes of codes and their pair (or 16
// bytes of bf16) on the cache's side, 16 bytes on the rows'. Bound by memory: store and load of 65536 rows of 8 heads of
// 128 with 8 bits in 135 us, 6.09 TB/s or 93 % of a copy's rate; of 512 rows in 4.3 us, two launches.
template <int D, int BITS, bool STORE, int HPT>
__global__ void __launch_bounds__(256) kv_copy_kernel(const __grid_constant__ CopyArgs A) {
  constexpr int LPH = D / 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int is_v = blockIdx.x >= A.deal[1].first;
  const Deal& deal = A.deal[is_v];
  const int l = threadIdx.x % LPH;
  uint32_t m0, tl;
  int chunk;
  const bool mine = dealt<LPH>(deal, m0, tl, chunk);
  const int h0 = HPT * chunk;
  const int n = min(HPT, A.kv.kv_heads - h0);
  uint32_t m = m0 + tl;
  const uint8_t* rows0 = A.rows[is_v] + h0 * (D * 2) + l * 16;
  const uint8_t* cache0 = at(is_v ? A.kv.v : A.kv.k, h0, A.kv.head_bytes) + l * (BITS == 16 ? 16 : 8);
  const uint8_t* pairs0 = at(is_v ? A.kv.vs : A.kv.ks, h0, A.kv.shead_bytes) + (l >> 3) * 4;
  int64_t s = m < A.M ? __ldg(A.slots + m) : -1;
  for (; m0 < A.M; m0 += deal.step, m += deal.step) {
    const bool live = mine && m < A.M;
    uint8_t* rows = at(rows0, live ? m : 0, A.stride[is_v]);
    uint4 raw[HPT];
    if (STORE) {
#pragma unroll
      for (int i = 0; i < HPT; ++i) {
        if (i > 0) { raw[i] = make_uint4(0, 0, 0, 0); }
        if (i == 0 || i < n) { raw[i] = ldg_stream_v4(rows + i * (D * 2)); }
      }
    }
    const bool there = s >= 0 && s < A.num_slots;
    if (live && s >= A.num_slots && l == 0) { atomicOr(A.status, kBadSlot); }
    uint32_t page = 0, place = 0;
    if (there) { split_slot(s, A.kv, page, place); }
    s = m + deal.step < A.M ? __ldg(A.slots + m + deal.step) : -1;  // of the next token
    uint8_t* cache = at(cache0 + page * A.kv.page_bytes, place, A.kv.token_bytes);
    uint8_t* pairs = at(pairs0 + page * A.kv.spage_bytes, place, A.kv.stoken_bytes);
    if (STORE) {
      const int writes = live && there ? n : 0;
#pragma unroll
      for (int i = 0; i < HPT; ++i) {
        if (BITS == 16) {
          if (i < writes) { *reinterpret_cast<uint4*>(cache + i * A.kv.head_bytes) = raw[i]; }
        } else {
          uint32_t pair;
          const uint2 c = quant8(raw[i], pair);
          if (i < writes) {
            *reinterpret_cast<uint2*>(cache + i * A.kv.head_bytes) = c;
            if ((l & 7) == 0) { *reinterpret_cast<uint32_t*>(pairs + i * A.kv.shead_bytes) = pair; }
          }
        }
      }
    } else {
      using Off = std::conditional_t<(HPT > 4), uint64_t, uint32_t>;  // four heads' offsets fit 32 bits (kv_check)
      uint32_t pair[HPT];
      const int reads = live && there ? n : 0;
#pragma unroll
      for (int i = 0; i < HPT; ++i) {
        pair[i] = 0;  // scale and bias 0: the value 0
        raw[i] = make_uint4(0, 0, 0, 0);
        if (i < reads) {
          if (BITS == 16) {
            raw[i] = *reinterpret_cast<const uint4*>(cache + i * A.kv.head_bytes);
          } else {
            const uint2 c = *reinterpret_cast<const uint2*>(cache + (Off)i * A.kv.head_bytes);
            raw[i].x = c.x, raw[i].y = c.y;
            pair[i] = *reinterpret_cast<const uint32_t*>(pairs + (Off)i * A.kv.shead_bytes);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < HPT; ++i) {
        if (BITS == 8) {
          const float sc = __uint_as_float(pair[i] << 16), b = __uint_as_float(pair[i] & 0xffff0000u);
          float x[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // 2^23 + code is a float with the code in its low byte
            x[e] = __fmaf_rn(sc, __fsub_rn(__uint_as_float(__byte_perm(raw[i].x, 0x4B000000u, 0x7650 | e)), 8388608.0f), b);
            x[4 + e] = __fmaf_rn(sc, __fsub_rn(__uint_as_float(__byte_perm(raw[i].y, 0x4B000000u, 0x7650 | e)), 8388608.0f), b);
          }
          raw[i] = pack8(x);
        }
        if (live && i < n) { *reinterpret_cast<uint4*>(rows + i * (D * 2)) = raw[i]; }
      }
    }
  }
}

bool strides_ok(int64_t s, int64_t mult) { return s >= 0 && s % mult == 0; }

// One head per lane group while the launch is too small to fill the machine (a decode step lives by
// latency), four once there are waves of them. Measured, one against four: one token 1.8 against 2.3 us, with an 8-bit
// store 2.3 against 3.3; 2048 tokens of 32 + 8 heads 20.4 against 12.4, 65536 rows through an 8-bit cache 176 against 135.
// (Two: 13.9 and 144; eight: 14.4 and 133, of which the loads' part is taken below.)
bool is_wide(int64_t M, int heads, int D, int sms) { return M * heads > (int64_t)sms * 8 * (256 / (D / 8)) * 2; }

struct Launch {
  dim3 grid, block;
};
// Deals `parts` parts of heads[] heads each. The blocks of all parts together are enough for `waves` times what the SMs
// hold at 64 registers a thread, shared out by the parts' chunks, those of k and v counted `costly` times.
// Measured, half as many waves / this / no limit: norm and rotation of 16320 tokens (4 waves) 108.5 / 106.7 / 113.3 us, 65536
// rows through an 8-bit cache (8 waves) 139 / 135 / 140. Rows into a cache cost more than query rows (slot, quantizer) and
// their blocks come last; counted once / twice: 8191 tokens of 32 + 8 + 8 heads of 128 into 16 bits 38.1 / 36.3 us, into 8 bits
// 41.6 / 39.4 (three times: 39.5); of 16 + 2 + 2 heads of 256 into 8 bits 39.6 / 37.9 (shared out by heads, not chunks: 44.8).
void deal(int64_t M, const int* heads, int parts, int hpt, int waves, int D, int sms, int costly, Deal* deals, Launch* l) {
  auto weight = [&](int part) { return part > 0 ? costly : 1; };
  const int groups = 256 / (D / 8);
  int total = 0, threads = 32;
  uint32_t first = 0;
  for (int i = 0; i < parts; ++i) {
    Deal& d = deals[i];
    d.chunks = (heads[i] + hpt - 1) / hpt;
    d.token_blocks = (d.chunks + groups - 1) / groups;
    d.per_block = (d.chunks + d.token_blocks - 1) / d.token_blocks;
    d.tokens = groups / d.per_block;
    // few tokens: spread them
    if (d.token_blocks > 1 || M < sms) { d.tokens = 1; }
    d.rcp = (65536u + d.per_block - 1) / d.per_block;
    total += d.chunks * weight(i);
    threads = std::max(threads, d.tokens * d.per_block * (D / 8));
  }
  threads = (threads + 31) & ~31;
  for (int i = 0; i < parts; ++i) {
    Deal& d = deals[i];
    const int64_t need = (M + d.tokens - 1) / d.tokens;
    const int64_t cap = (int64_t)sms * (1024 / threads) * waves * (d.chunks * weight(i)) / total / d.token_blocks;
    const int64_t blocks = std::min(need, std::max<int64_t>(cap, 1));
    d.first = first;
    d.step = (uint32_t)(blocks * d.tokens);
    first += (uint32_t)(blocks * d.token_blocks);
  }
  l->block = dim3((unsigned)threads);
  l->grid = dim3(first);
}

template <typename K, typename A>
int launch_with_pdl(K kern, const Launch& d, cudaStream_t st, const A& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = d.grid;
  cfg.blockDim = d.block;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VPQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a));
  return VPQ_OK;
}

template <int MODE>
int launch_norm(const QkArgs& a0, int D, cudaStream_t st) {
  QkArgs a = a0;
  Launch l;
  const int sms = num_sms();
  const bool wide = is_wide(a.M, a.heads[0] + (MODE ? 2 : 1) * a.heads[1], D, sms);
  deal(a.M, a.heads, MODE ? 3 : 2, wide ? 4 : 1, 4, D, sms, MODE ? 2 : 1, a.deal, &l);
  if (D == 64) {
    return wide ? launch_with_pdl(norm_rope_store_kernel<64, MODE, 4>, l, st, a)
                : launch_with_pdl(norm_rope_store_kernel<64, MODE, 1>, l, st, a);
  }
  if (D == 128) {
    return wide ? launch_with_pdl(norm_rope_store_kernel<128, MODE, 4>, l, st, a)
                : launch_with_pdl(norm_rope_store_kernel<128, MODE, 1>, l, st, a);
  }
  return wide ? launch_with_pdl(norm_rope_store_kernel<256, MODE, 4>, l, st, a)
              : launch_with_pdl(norm_rope_store_kernel<256, MODE, 1>, l, st, a);
}

template <int BITS, bool STORE>
int launch_copy(const CopyArgs& a0, int D, cudaStream_t st) {
  CopyArgs a = a0;
  Launch l;
  const int sms = num_sms();
  const bool wide = a.kv.kv_heads >= 4 && is_wide(a.M, 2 * a.kv.kv_heads, D, sms);
  // Codes come in half rows, so eight heads of them are as many bytes in flight as four of bf16. Loads of 8 bits, 8 heads,
  // eight against four at a time: D 128 65536 rows 63.4 against 69.2 us, D 64 131072 rows 63.7 against 69.4, D 256 32768 rows
  // 63.4 against 66.7. Stores, and loads of 16 bits, gain 1 % or lose as much.
  constexpr int kMost = BITS == 8 && !STORE ? 8 : 4;
  const bool most = wide && a.kv.kv_heads % kMost == 0;
  const int heads[2] = {a.kv.kv_heads, a.kv.kv_heads};
  deal(a.M, heads, 2, most ? kMost : (wide ? 4 : 1), 8, D, sms, 1, a.deal, &l);
#define VPQ_GO(DIM)                                                                                   \
  return most   ? launch_with_pdl(kv_copy_kernel<DIM, BITS, STORE, kMost>, l, st, a)                  \
         : wide ? launch_with_pdl(kv_copy_kernel<DIM, BITS, STORE, 4>, l, st, a)                      \
                : launch_with_pdl(kv_copy_kernel<DIM, BITS, STORE, 1>, l, st, a);
  if (D == 64) { VPQ_GO(64) }
  if (D == 128) { VPQ_GO(128) }
  VPQ_GO(256)
#undef VPQ_GO
}

bool known_dim(int d) { return d == 64 || d == 128 || d == 256; }

// Fills and checks one row operand; stride 0 = dense.
int take_rows(const char* who, const char* name, const void* p, int64_t stride, int64_t heads, int D, uint32_t* bytes) {
  if (!p) { return fail(VPQ_ERR_INVALID_ARG, "%s: %s is null", who, name); }
  if (stride == 0) { stride = heads * D; }
  if (stride < heads * D) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: %s rows overlap (stride %lld for %lld values)", who, name, (long long)stride,
                (long long)(heads * D));
  }
  if (stride > INT_MAX / 2) { return fail(VPQ_ERR_INVALID_ARG, "%s: the rows of %s are 2^31 bytes or more apart", who, name); }
  if (!aligned16(p) || (stride & 7)) {
    return fail(VPQ_ERR_ALIGNMENT, "%s: %s and its row stride must be multiples of 16 bytes", who, name);
  }
  *bytes = (uint32_t)(stride * 2);
  return VPQ_OK;
}

// The part of a vpq_qk_desc that both entry points share.
int take_qk(const char* who, const vpq_qk_desc& d, QkArgs* a) {
  if (d.M <= 0 || d.q_heads <= 0 || d.kv_heads <= 0) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: need M>0, q_heads>0, kv_heads>0 (M=%lld q_heads=%d kv_heads=%d)", who,
                (long long)d.M, d.q_heads, d.kv_heads);
  }
  if (!known_dim(d.head_dim)) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256 (got %d)", who, d.head_dim);
  }
  if (d.q_heads > 65536 || d.kv_heads > 65536 || d.M > INT_MAX / 2) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: at most 65536 heads and 2^30 rows", who);
  }
  if (d.cos_sin) {
    if (d.rot_dim <= 0 || d.rot_dim > d.head_dim || (d.rot_dim & 15)) {
      return fail(VPQ_ERR_INVALID_ARG, "%s: rot_dim must be a multiple of 16 up to head_dim (rot_dim=%d head_dim=%d)", who,
                  d.rot_dim, d.head_dim);
    }
    if (d.table_rows <= 0 || (!d.positions && d.table_rows < d.M)) {
      return fail(VPQ_ERR_INVALID_ARG, "%s: cos_sin has %lld rows, %lld are needed", who, (long long)d.table_rows,
                  (long long)(d.positions ? 1 : d.M));
    }
    if (!aligned16(d.cos_sin) || (reinterpret_cast<uintptr_t>(d.positions) & 3)) {
      return fail(VPQ_ERR_ALIGNMENT, "%s: cos_sin must be 16-byte aligned, positions 4-byte", who);
    }
  } else if (d.rot_dim != 0 || d.positions) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: rot_dim and positions need cos_sin", who);
  }
  if (!(d.eps >= 0.0f)) { return fail(VPQ_ERR_INVALID_ARG, "%s: eps must not be negative", who); }
  if (!aligned16(d.q_norm_w) || !aligned16(d.k_norm_w)) {
    return fail(VPQ_ERR_ALIGNMENT, "%s: norm weights must be 16-byte aligned", who);
  }
  a->norm_w[0] = static_cast<const uint16_t*>(d.q_norm_w);
  a->norm_w[1] = static_cast<const uint16_t*>(d.k_norm_w);
  a->cos_sin = d.cos_sin;
  a->positions = d.positions;
  a->M = (uint32_t)d.M;
  a->table_rows = (uint32_t)std::min<int64_t>(d.table_rows, INT_MAX);  // positions name no more
  a->heads[0] = d.q_heads;
  a->heads[1] = d.kv_heads;
  a->heads[2] = d.kv_heads;
  a->rot = d.rot_dim;
  a->interleaved = d.interleaved != 0;
  a->eps = d.eps;
  a->inv_d = 1.0f / (float)d.head_dim;
  if (int rc = take_rows(who, "q", d.q, d.q_stride, d.q_heads, d.head_dim, &a->in_stride[0])) { return rc; }
  if (int rc = take_rows(who, "k", d.k, d.k_stride, d.kv_heads, d.head_dim, &a->in_stride[1])) { return rc; }
  if (int rc = take_rows(who, "q_out", d.q_out, d.q_out_stride, d.q_heads, d.head_dim, &a->out_stride[0])) { return rc; }
  a->in[0] = static_cast<const uint8_t*>(d.q);
  a->in[1] = static_cast<const uint8_t*>(d.k);
  a->out[0] = static_cast<uint8_t*>(d.q_out);
  if (d.q_out == d.q && a->out_stride[0] != a->in_stride[0]) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: q_out is q with another row stride", who);
  }
  return VPQ_OK;
}

int take_slots(const char* who, const int64_t* slots) {
  if (!slots) { return fail(VPQ_ERR_INVALID_ARG, "%s: slots is null", who); }
  if (reinterpret_cast<uintptr_t>(slots) & 7) { return fail(VPQ_ERR_ALIGNMENT, "%s: slots must be 8-byte aligned", who); }
  return VPQ_OK;
}

}  // namespace

int kv_check(const char* who, const vpq_kv_cache* c, KvView* view) {
  if (!c) { return fail(VPQ_ERR_INVALID_ARG, "%s: null cache", who); }
  if (c->bits != 8 && c->bits != 16) { return fail(VPQ_ERR_UNSUPPORTED, "%s: a cache has 16 or 8 bits (got %d)", who, c->bits); }
  if (!known_dim(c->head_dim)) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256 (got %d)", who, c->head_dim);
  }
  if (c->num_pages <= 0 || c->num_pages > INT_MAX || c->kv_heads <= 0 || c->kv_heads > 65536) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: need 0 < num_pages < 2^31, 0 < kv_heads <= 65536 (num_pages=%lld kv_heads=%d)", who,
                (long long)c->num_pages, c->kv_heads);
  }
  if (c->page_size <= 0 || (c->page_size & 15) || c->page_size > (1 << 20)) {
    return fail(VPQ_ERR_UNSUPPORTED, "%s: page_size must be a multiple of 16, at most 2^20 (got %d)", who, c->page_size);
  }
  const bool q = c->bits == 8;
  if (!c->k || !c->v || (q && (!c->k_scales || !c->v_scales))) { return fail(VPQ_ERR_INVALID_ARG, "%s: null pages", who); }
  if (!q && (c->k_scales || c->v_scales)) { return fail(VPQ_ERR_INVALID_ARG, "%s: a 16-bit cache has no scales", who); }
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scales) || !aligned16(c->v_scales)) {
    return fail(VPQ_ERR_ALIGNMENT, "%s: pages and scales must be 16-byte aligned", who);
  }
  const int64_t D = c->head_dim, elt = q ? 1 : 2;
  int64_t ps = c->page_stride, hs = c->head_stride, ts = c->token_stride;
  if (!ps && !hs && !ts) { ts = D, hs = ts * c->page_size, ps = hs * c->kv_heads; }
  const int64_t pairs = D / kKvGroup * 2;
  int64_t sps = c->scale_page_stride, shs = c->scale_head_stride, sts = c->scale_token_stride;
  if (!sps && !shs && !sts) { sts = pairs, shs = sts * c->page_size, sps = shs * c->kv_heads; }
  if (ts < D || (hs < D && c->kv_heads > 1) || (ps < D && c->num_pages > 1) || hs < 0 || ps < 0 ||
      (q && (sts < pairs || (shs < pairs && c->kv_heads > 1) || (sps < pairs && c->num_pages > 1) || shs < 0 || sps < 0))) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: a stride is smaller than a row", who);
  }
  // the stride of the only head or page does not matter
  if (c->kv_heads == 1) { hs = shs = 0; }
  if (c->num_pages == 1) { ps = sps = 0; }
  const int64_t lim = INT_MAX / 2 / elt, slim = INT_MAX / 2 / 2;  // four heads' offsets in bytes fit 32 bits
  if (ts > lim || hs > lim || sts > slim || shs > slim || ps > ((int64_t)1 << 46) / c->num_pages ||
      sps > ((int64_t)1 << 46) / c->num_pages) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: a stride is out of range (token and head strides stay below 2^30 bytes)", who);
  }
  const int64_t mult = 16 / elt;
  if (!strides_ok(ts, mult) || !strides_ok(hs, mult) || !strides_ok(ps, mult) ||
      (q && (!strides_ok(sts, pairs) || !strides_ok(shs, pairs) || !strides_ok(sps, pairs)))) {
    return fail(VPQ_ERR_ALIGNMENT, "%s: page strides must be multiples of 16 bytes, scale strides of head_dim / 32", who);
  }
  view->k = static_cast<uint8_t*>(c->k);
  view->v = static_cast<uint8_t*>(c->v);
  view->ks = static_cast<uint8_t*>(c->k_scales);
  view->vs = static_cast<uint8_t*>(c->v_scales);
  view->num_pages = c->num_pages;
  view->page_bytes = ps * elt;
  view->head_bytes = (uint32_t)(hs * elt);
  view->token_bytes = (uint32_t)(ts * elt);
  view->spage_bytes = sps * 2;
  view->shead_bytes = (uint32_t)(shs * 2);
  view->stoken_bytes = (uint32_t)(sts * 2);
  view->page_size = c->page_size;
  view->page_shift = -1;
  for (int s = 4; s <= 20; ++s) {
    if (c->page_size == (1 << s)) { view->page_shift = s; }
  }
  view->kv_heads = c->kv_heads;
  return VPQ_OK;
}

}  // namespace vpq

using namespace vpq;

extern "C" int vpq_qk_norm_rope_bf16(const vpq_qk_desc* desc_host, void* stream) {
  const char* who = "qk_norm_rope";
  clear_error();
  if (!desc_host) { return fail(VPQ_ERR_INVALID_ARG, "%s: null descriptor", who); }
  QkArgs a = {};
  if (int rc = take_qk(who, *desc_host, &a)) { return rc; }
  if (int rc = take_rows(who, "k_out", desc_host->k_out, desc_host->k_out_stride, desc_host->kv_heads, desc_host->head_dim, &a.out_stride[1])) {
    return rc;
  }
  a.out[1] = static_cast<uint8_t*>(desc_host->k_out);
  if (desc_host->k_out == desc_host->k && a.out_stride[1] != a.in_stride[1]) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: k_out is k with another row stride", who);
  }
  if (int rc = require_sm100()) { return rc; }
  if (int rc = index_status_word(&a.status)) { return rc; }
  return launch_norm<0>(a, desc_host->head_dim, static_cast<cudaStream_t>(stream));
}

extern "C" int vpq_qkv_norm_rope_store_bf16(const vpq_qk_desc* desc_host, const vpq_kv_cache* cache_host,
                                            const int64_t* slots, void* stream) {
  const char* who = "qkv_norm_rope_store";
  clear_error();
  if (!desc_host) { return fail(VPQ_ERR_INVALID_ARG, "%s: null descriptor", who); }
  QkArgs a = {};
  if (int rc = take_qk(who, *desc_host, &a)) { return rc; }
  if (int rc = take_rows(who, "v", desc_host->v, desc_host->v_stride, desc_host->kv_heads, desc_host->head_dim, &a.in_stride[2])) {
    return rc;
  }
  a.in[2] = static_cast<const uint8_t*>(desc_host->v);
  if (int rc = kv_check(who, cache_host, &a.kv)) { return rc; }
  if (cache_host->kv_heads != desc_host->kv_heads || cache_host->head_dim != desc_host->head_dim) {
    return fail(VPQ_ERR_INVALID_ARG, "%s: the cache has %d heads of %d, the rows %d of %d", who, cache_host->kv_heads,
                cache_host->head_dim, desc_host->kv_heads, desc_host->head_dim);
  }
  if (int rc = take_slots(who, slots)) { return rc; }
  a.slots = slots;
  a.num_slots = a.kv.num_pages * a.kv.page_size;
  if (int rc = require_sm100()) { return rc; }
  if (int rc = index_status_word(&a.status)) { return rc; }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache_host->bits == 8 ? launch_norm<8>(a, desc_host->head_dim, st)
                               : launch_norm<16>(a, desc_host->head_dim, st);
}

namespace {
template <bool STORE>
int copy_rows(const char* who, const vpq_kv_cache* c, const void* k, const void* v, int64_t k_stride, int64_t v_stride,
              const int64_t* slots, int64_t M, void* stream) {
  clear_error();
  CopyArgs a = {};
  if (int rc = kv_check(who, c, &a.kv)) { return rc; }
  if (M <= 0) { return fail(VPQ_ERR_INVALID_ARG, "%s: need M > 0 (M=%lld)", who, (long long)M); }
  if (M > INT_MAX / 2) { return fail(VPQ_ERR_UNSUPPORTED, "%s: at most 2^30 rows (M=%lld)", who, (long long)M); }
  const int D = c->head_dim, H = c->kv_heads;
  if (int rc = take_rows(who, STORE ? "k" : "k_out", k, k_stride, H, D, &a.stride[0])) { return rc; }
  if (int rc = take_rows(who, STORE ? "v" : "v_out", v, v_stride, H, D, &a.stride[1])) { return rc; }
  if (int rc = take_slots(who, slots)) { return rc; }
  a.rows[0] = static_cast<uint8_t*>(const_cast<void*>(k));
  a.rows[1] = static_cast<uint8_t*>(const_cast<void*>(v));
  a.slots = slots;
  a.M = (uint32_t)M;
  a.num_slots = a.kv.num_pages * a.kv.page_size;
  if (int rc = require_sm100()) { return rc; }
  if (int rc = index_status_word(&a.status)) { return rc; }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return c->bits == 8 ? launch_copy<8, STORE>(a, D, st) : launch_copy<16, STORE>(a, D, st);
}
}  // namespace

extern "C" int vpq_kv_store_bf16(const vpq_kv_cache* cache_host, const void* k, const void* v, int64_t k_stride,
                                 int64_t v_stride, const int64_t* slots, int64_t M, void* stream) {
  return copy_rows<true>("kv_store", cache_host, k, v, k_stride, v_stride, slots, M, stream);
}

extern "C" int vpq_kv_load_bf16(const vpq_kv_cache* cache_host, void* k_out, void* v_out, int64_t k_stride,
                                int64_t v_stride, const int64_t* slots, int64_t M, void* stream) {
  return copy_rows<false>("kv_load", cache_host, k_out, v_out, k_stride, v_stride, slots, M, stream);
}
