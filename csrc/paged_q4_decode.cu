// Attention of single query rows over the 4-bit paged cache (format: q4.cuh) on sm_100a.
//
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q . k_t),  k_td = sk_tg (n_td - 8),  v_td = sv_tg (m_td - 8)
//
// Up to eight query heads of a kv head's group are the N dimension of mma.sync.m16n8k16 (fp16, fp32 sums), 16 tokens the M
// dimension of K Q^T and 16 elements that of V^T P^T: every row of the matrix instructions is used.
//   * A code needs no conversion: four bits at the bottom of an fp16 are the number n 2^-24, exact in the matrix
//     instruction, so a word & 0x000f000f is two operands, & 0x00f000f0 two more that are 16 n 2^-24; shifted by 8 the word gives
//     the other four. The factor 16 is taken out of the query elements beforehand. Values are rows of the product, which may be
//     any combinations of elements that can be solved for: n and n + 16 n', the lower and the upper bytes of the word as they
//     are, which saves an instruction in five; n' is had from the two sums at the end, to 2^-18 of the row's magnitude.
//   * q . (n - 8) = q . n - 8 sum q: the second part is a product of the key scales with a constant of the query, one matrix
//     instruction for all groups (the constant as fp16 plus what fp16 leaves of it, 22 bits). On the value side another one,
//     whose constant operand has -8 in row g, sums -8 p_t sv_tg from the same rounded products.
//   * The scale of a group multiplies a finished dot product (keys) or the probability before it is rounded to fp16 (values).
//   * Queries are scaled per head by a power of two to [2^14, 2^15) so that bf16 fits fp16: an element loses bits only below
//     2^-24 of the head's largest.
//   * p_t sv_tg is rounded to fp16 too. Its range is held by the maximum that the softmax subtracts: it runs over
//     log2 p_t + log2 max_g |sv_tg| instead of log2 p_t, so that the largest product is 2^12 to 2^15, whatever the values'
//     magnitude. Relative error 2^-11 down to 2^-26 of the largest contribution of any group of the head (a token whose values in
//     one group are 2^20 times those elsewhere costs the other groups bits); sums, maxima and p itself stay in fp32.
//   * Scores may have any size: from 2^22 on a maximum in fp32 does not do, and dot products are compared instead (Q4State).
// Tokens outside the sequence get probability and value scale zero by selection, so nothing stale in a page (NaN scales
// included) reaches a result. A page number outside the pool counts as a page outside the sequence.
//
// Two kernels. One block per (row, slice of heads) where the table is narrow (q4_unit_warps); else all tiles of the call in one
// line, cut evenly over the warps that the GPU holds, and a second kernel that joins the parts (Q4Plan).
//
// Bounds. The bytes are 4.5 bits an element, each read once: at the copy bandwidth an SM gets a tile of 2304 bytes in about
// 100 clocks, in which its four schedulers can issue 400 instructions; a tile takes about 310, of them 72 to unpack 4096 codes
// and 21 matrix instructions (0.28 of their pipe). With 128 registers a thread, 16 warps on an SM issue 0.57 of the slots: the
// kernels are held by the latencies of dependent instructions, not by memory. Captured calls over caches larger than L2, beside
// the attention over the 16-bit cache: 512 rows of 768 tokens, 12 heads on 2 of 128, 28.8 us, 0.60 of the copy bandwidth (16 bits:
// 109 us); 64 rows of 2000, 32 on 32, 103 us, 0.88 (391); 4 rows of 100000, 32 on 8, 86.6 us, 0.81 (381); 33 rows of up to 1500,
// 12 on 12 of 64, 11.2 us (40); one row of 333, 5.5 us (9.6). Heads of 192 and 256 need up to 255 registers a thread: eight warps on
// an SM hide the same latencies (64 rows of 4000, 8 on 1 of 256, 28.1 us, 0.40; of 192, 23.7, 0.36; of 1000 and 256, 13.6, 0.21).
#include <math.h>
#include <string.h>

#include "host_common.h"
#include "launch_behind.cuh"
#include "ptx.cuh"
#include "q4.cuh"

namespace icb {

constexpr int kQ4Warps = 4;
constexpr int kQ4Threads = kQ4Warps * 32;
// Least tiles of a warp: with fewer, joining the parts of a long row among short ones takes longer than what it gains. With 2, 6 and
// 12, us: one row of 8000 tokens among 255 of 100 (12 heads on 2, a table of 20000: in a table of 8000 it does not come here) 43.8,
// 24.9, 24.7; 4 rows of 4000 (32 on 8) 15.8, 15.4, 16.2; 16 of 8000 (12 on 2) 20.7, 20.7, 21.0.
constexpr int kQ4MinTiles = 6;
constexpr int kQ4Whole = 8;                     // units of at most so many tiles are not divided among warps
constexpr float kQ4Top = 12.f;                  // log2 of the largest fp16 probability times scale right after a new maximum
constexpr float kQ4Limit = 32768.f;             // and what it may grow to before the maximum is taken again: fp16 holds it
constexpr float kQ4None = 3e38f, kQ4Far = 2e38f;            // Q4State::off of no tokens, and of scores from kQ4Large on
constexpr float kQ4Large = 4194304.f;           // 2^22: up to here a maximum in fp32 is within 1/2 of itself
constexpr int kQ4MostFactor = 99;               // log2 of the largest factor from dot products to scores (its mantissa apart)
constexpr float kLog2e = 1.4426950408889634f;

struct Q4DecodeArgs {
  const uint16_t* q;
  long long q_stride;
  const uint8_t* pool;
  const int* block_table;
  const int* seqs;              // or null
  const int* lens;
  uint16_t* out;                // [rows, out_stride], heads HD apart
  long long out_stride;
  int4* owner;                  // {row, unit, first, last worker} of a unit that several warps share, or row -1; one entry for
  int by_unit;                  // each unit of the call, or (by_unit 0) for each warp: the unit that begins in its range
  float* part;                  // [workers][2][slice heads] records of HD + 4 floats: outputs, Q4State::end
  int rows, hq, hkv, slices, heads, tiles, max_blocks, table_rows, num_blocks;   // heads: of a slice, at most eight
  int workers;                  // warps that share the tiles
  float scale;                  // score factor times log2(e) without its power of two (0, or 0.7 to 1.5), the exponent of that
  int scale_exp;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(global) : "memory");
}

// A tile (NG * 576 bytes) to shared memory, this lane's 16 of every 512 bytes; nothing if `there` is false.
template <int NG>
__device__ __forceinline__ void copy_tile(uint32_t smem, const uint8_t* global, bool there) {
  constexpr int FULL = NG * 576 / 512;
#pragma unroll
  for (int i = 0; i < FULL; ++i)
    asm volatile("{ .reg .pred p; setp.ne.s32 p, %2, 0; @p cp.async.cg.shared.global [%0], [%1], 16; }" ::"r"(smem + i * 512),
                 "l"(global + i * 512), "r"((int)there) : "memory");
  if (NG * 576 % 512 != 0)
    asm volatile("{ .reg .pred p; setp.ne.s32 p, %2, 0; @p cp.async.cg.shared.global [%0], [%1], 16; }" ::"r"(smem + FULL * 512),
                 "l"(global + FULL * 512), "r"((int)(there && (threadIdx.x & 31) * 16 < NG * 576 % 512)) : "memory");
}

template <bool BF16>
__device__ __forceinline__ void q4_store4(uint16_t* to, float x, float y, float z, float w) {
  // rows of any pitch and alignment
  const float v[4] = {x, y, z, w};
  if ((reinterpret_cast<uintptr_t>(to) & 7) == 0) {
    *reinterpret_cast<uint2*>(to) = BF16 ? make_uint2(pack_bf16x2(x, y), pack_bf16x2(z, w))
                                         : make_uint2(pack_f16x2(x, y), pack_f16x2(z, w));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) reinterpret_cast<__nv_bfloat16*>(to)[i] = __float2bfloat16(v[i]);
    else reinterpret_cast<__half*>(to)[i] = __float2half(v[i]);
  }
}

// The query operand, resident in registers: column n of the matrix instructions is head n (T = 1, up to eight heads) or head
// n & 3 (T = 2, up to four: columns 4 .. 7 are the same heads for a second tile).
template <int NG, int T>
struct Q4Query {
  uint32_t b[NG][4];            // B fragments of the two matrix instructions of a group
  // -8 * sum of each group's elements, in the units of the dot products (2^-24). T = 1: the B fragment of a product over the
  // groups, as fp16 and what it leaves (out of that, below 2^-15 of a step of the largest element). T = 2, where a product would
  // need the scales of two tiles: columns 2c, 2c + 1
  uint32_t starts[NG > 4 ? 2 : 1];
  float start[T == 2 ? NG : 1][2];
  float factor[2];              // from the dot products to the base-2 score
};

template <int NG, int T, bool BF16>
__device__ __forceinline__ void q4_load_query(Q4Query<NG, T>& f, const uint8_t* q, int heads, float scale, int scale_exp) {
  constexpr int HD = NG * 32;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, head = T == 1 ? r : r & 3;
  float x[NG][8];
  float top = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (head < heads) u = *reinterpret_cast<const uint4*>(q + (head * HD + g * 32 + c * 8) * 2);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = BF16 ? unpack_bf16x2(w[i]) : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[g][2 * i] = t.x;
      x[g][2 * i + 1] = t.y;
      top = fmaxf(top, fmaxf(fabsf(t.x), fabsf(t.y)));
    }
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (BF16 && __any_sync(0xffffffffu, top > 0.f && top < 5.4210109e-20f)) {     // below 2^-64: `up` alone may not reach
    const bool lift = top < 5.4210109e-20f;
    scale_exp -= lift ? 64 : 0;
    top *= lift ? 18446744073709551616.f : 1.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[g][i] *= lift ? 18446744073709551616.f : 1.f;
    }
  }
  const int e = min(max((__float_as_int(top) >> 23) - 127, -100), 127);
  const float up = copysignf(__int_as_float((127 + 14 - e) << 23), scale), up16 = up * 0.0625f;
  // 2^24 / up * scale, which must send the -infinity of a masked score to itself: positive, the query having the sign of the scale.
  // Dot products are multiples of 2^-72 (2^-24 each of the query, the code, the scale) below 2^18, so that beyond 2^99 a larger
  // factor changes nothing: scores that differ at all do so by 2^27, and none is an infinity
  const int back_exp = min(max(10 + e + scale_exp, -126), kQ4MostFactor);
  const float back = fmaxf(__int_as_float((127 + back_exp) << 23) * fabsf(scale), 1.17549435e-38f);
  float own[NG > 4 ? 2 : 1] = {};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float sum = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m) {                                            // elements 2m, 2m + 4 and 2m + 1, 2m + 5
      const __half2 even = __floats2half2_rn(x[g][2 * m] * up, x[g][2 * m + 4] * up);
      const __half2 odd = __floats2half2_rn(x[g][2 * m + 1] * up16, x[g][2 * m + 5] * up16);
      f.b[g][2 * m] = *reinterpret_cast<const uint32_t*>(&even);
      f.b[g][2 * m + 1] = *reinterpret_cast<const uint32_t*>(&odd);
      const float2 fe = __half22float2(even), fo = __half22float2(odd);
      sum += fe.x + fe.y + 16.f * (fo.x + fo.y);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    sum *= -8.f / 16777216.f;
    if (T == 1) {
      if ((g & 3) == c) own[g >> 2] = sum;                                   // k slots 2c, 2c + 1 belong to group c (and c + 4)
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) f.start[g][i] = __shfl_sync(0xffffffffu, sum, 8 * c + 4 * i);  // column 2c + i: lanes 4 (2c + i) ..
    }
  }
  if (T == 1) {
#pragma unroll
    for (int i = 0; i < (NG > 4 ? 2 : 1); ++i) {
      const __half hi = __float2half_rn(own[i]);
      const __half2 both = __halves2half2(hi, __float2half_rn(own[i] - __half2float(hi)));
      f.starts[i] = *reinterpret_cast<const uint32_t*>(&both);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) f.factor[i] = __shfl_sync(0xffffffffu, back, 8 * c + 4 * i);
}

// Sums of several parts over tokens, each with its own {at, off} (Q4State): the one to bring them to is that of the largest
// maximum (either of two that fp32 does not tell apart), and what a part is to be multiplied with.
__device__ __forceinline__ float2 q4_larger(const float2& a, const float2& b, float factor) {
  return fmaf(b.x, factor, -b.y) > fmaf(a.x, factor, -a.y) ? b : a;
}
__device__ __forceinline__ float q4_weight(const float2& part, const float2& all, float factor) {
  return exp2_fast(fmaf(part.x - all.x, factor, all.y - part.y));
}
__device__ __forceinline__ float2 q4_from(const float2& x, int half) {         // of the lane with this bit 1
  const int lane = (threadIdx.x & 29) | half;
  return make_float2(__shfl_sync(0xffffffffu, x.x, lane), __shfl_sync(0xffffffffu, x.y, lane));
}

// Running state of a warp: this lane's part of eight columns. Of a dot product s, p = exp2((s - at) * factor + off). `at` is 0 as
// long as the largest score is below kQ4Large. From there on a maximum rounded to fp32 would lie too far from the score it is
// to be subtracted from (by 32 at 2^30: p of 2^32 or 2^-32), so `at` is the largest dot product, whose distance to others is
// exact enough, and `off` stays small: both are in shared memory, and kQ4Far for an `off` sends every pass there. That such
// scores may come costs others little (512 rows of 768 tokens 29.0 -> 29.2 us, 78 of 264 11.9 -> 12.5); subtracting `at` in every
// pass took 3 % more for the 512 rows.
template <int NG>
struct Q4State {
  float o[NG][2][4];            // V^T P^T: elements 32 g + 4 r + 2 m + (reg >> 1), columns 2c + (reg & 1); odd elements times
                                // 16 and with the even one below added
  float z[4];                   // row g: -8 * sum of the rounded p * value scale of group g, in the units of o (even elements)
  float off[2], l[2];           // of columns 2c, 2c + 1 (equal in all lanes r); sum of this lane's p
  float2* far;                  // this lane's {at, off} of both where `off` is kQ4Far
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[g][0][i] = o[g][1][i] = 0.f;
    }
    z[0] = z[1] = z[2] = z[3] = 0.f;
    off[0] = off[1] = kQ4None;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ float2 place(int e) const { return off[e] == kQ4Far ? far[e] : make_float2(0.f, off[e]); }
  __device__ __forceinline__ void rescale(int e, float by) {
    l[e] *= by;
    z[e] *= by;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int t = 0; t < 2; ++t) { o[g][t][e] *= by; o[g][t][2 + e] *= by; }
    }
  }
  // The end of a part's record: {off, sum}, or {kQ4Far, sum, at, factor} with all sums of the column as for an `off` of 0.
  __device__ __forceinline__ float4 end(int e, float factor) {
    float at = 0.f;
    if (off[e] == kQ4Far) {
      at = far[e].x;
      rescale(e, exp2_fast(-far[e].y));
    }
    return make_float4(off[e], l[e], at, factor);
  }
  // Columns n and n + 4 hold the same head over different tokens: both become their sum.
  __device__ __forceinline__ void fold(const float (&factor)[2]) {
    const bool large = __any_sync(0xffffffffu, off[0] == kQ4Far || off[1] == kQ4Far);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (large) {
        const float2 mine = place(e), both = q4_larger(q4_from(mine, 0), q4_from(mine, 2), factor[e]);
        rescale(e, q4_weight(mine, both, factor[e]));
        off[e] = both.x != 0.f ? kQ4Far : both.y;
        far[e] = both;
      } else {
        const float next = fminf(off[e], __shfl_xor_sync(0xffffffffu, off[e], 2));
        rescale(e, exp2_fast(next - off[e]));
        off[e] = next;
      }
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      z[e] += __shfl_xor_sync(0xffffffffu, z[e], 2);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          o[g][t][e] += __shfl_xor_sync(0xffffffffu, o[g][t][e], 2);
          o[g][t][2 + e] += __shfl_xor_sync(0xffffffffu, o[g][t][2 + e], 2);
        }
      }
    }
  }
};

// T tiles of 16 tokens in shared memory, neighbours in the sequence. WHOLE: all of them belong to it; else `live` tokens do, bit
// j of `gone`: tile T - 1 - j is not there. (Heads over 128 always go the second way: another copy of their code costs more than
// the masks, 64 rows of 1000 tokens with heads of 256 take 16.6 us with it and 14.6 without.) With T = 2 both tiles go through
// the same columns' arithmetic at once: columns 0 .. 3 are the heads over the first tile, 4 .. 7 over the second, which a group of
// at most four heads would leave idle.
template <int NG, int T, bool WHOLE>
__device__ __forceinline__ void q4_pass(Q4State<NG>& st, const Q4Query<NG, T>& f, const uint8_t* tiles, int live,
                                        uint32_t gone) {
  constexpr int NP = NG / 2, TILE = 576 * NG;    // NP: 16-byte pieces per lane of the keys, and of the values
  const int lane = threadIdx.x & 31, r = lane >> 2, second = T == 2 ? (lane >> 1) & 1 : 0;
  // scales of tokens r and r + 8 of this lane's tile: NG fp16 of the keys, NG of the values
  uint32_t sc[2][NG];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint8_t* at = tiles + second * TILE + 512 * NG + (r + 8 * j) * 4 * NG;
    if (NG % 4 == 0) {
#pragma unroll
      for (int i = 0; i < NG / 4; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(at + 16 * i);
        sc[j][4 * i] = u.x; sc[j][4 * i + 1] = u.y; sc[j][4 * i + 2] = u.z; sc[j][4 * i + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NG / 2; ++i) {
        const uint2 u = *reinterpret_cast<const uint2*>(at + 8 * i);
        sc[j][2 * i] = u.x; sc[j][2 * i + 1] = u.y;
      }
    }
  }
  // ---- scores of tokens r, r + 8 and columns 2c, 2c + 1: s[2 j + e]
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (T == 1) {                                  // the part of the -8: key scales times `starts`
    const uint32_t pick = 0x1010u + 0x2222u * (NG == 2 ? lane & 1 : lane & 3);       // scale of group c, twice
    const uint32_t a0 = __byte_perm(sc[0][0], sc[0][NG == 2 ? 0 : 1], pick);
    const uint32_t a1 = __byte_perm(sc[1][0], sc[1][NG == 2 ? 0 : 1], pick);
    if (NG <= 4) {
      mma_f16_first(s, a0, a1, 0u, 0u, f.starts[0], 0u);
    } else {
      const uint32_t pick2 = 0x1010u + 0x2222u * (NG == 6 ? lane & 1 : lane & 3);    // and of group c + 4
      constexpr int K2 = NG > 4 ? 2 : 0, K3 = NG == 8 ? 3 : K2;
      mma_f16_first(s, a0, a1, __byte_perm(sc[0][K2], sc[0][K3], pick2), __byte_perm(sc[1][K2], sc[1][K3], pick2), f.starts[0],
                    f.starts[NG > 4 ? 1 : 0]);
    }
  }
  {
    uint32_t kw[T][2 * NG];
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const uint4 u = *reinterpret_cast<const uint4*>(tiles + t * TILE + p * 512 + lane * 16);
        kw[t][4 * p] = u.x; kw[t][4 * p + 1] = u.y; kw[t][4 * p + 2] = u.z; kw[t][4 * p + 3] = u.w;
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float d[T][4];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const uint32_t a = kw[t][g], b = kw[t][NG + g], a8 = a >> 8, b8 = b >> 8;
        mma_f16_first(d[t], a & 0x000f000fu, b & 0x000f000fu, a & 0x00f000f0u, b & 0x00f000f0u, f.b[g][0], f.b[g][1]);
        mma_f16(d[t], a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u, f.b[g][2], f.b[g][3]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&sc[j][g >> 1]));
        const float ks = (g & 1) ? two.y : two.x;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float dot = T == 2 && second ? d[T - 1][2 * j + e] : d[0][2 * j + e];
          s[2 * j + e] = fmaf(ks, T == 2 ? dot + f.start[T == 2 ? g : 0][e] : dot, s[2 * j + e]);
        }
      }
    }
  }
  if (!WHOLE) {
    const int mine = (gone >> (T - 1 - second) & 1) ? 0 : live - second * kQ4Tile;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (r + 8 * j < mine) continue;
      s[2 * j] = s[2 * j + 1] = -INFINITY;
#pragma unroll
      for (int g = NG / 2; g < NG; ++g) sc[j][g] = 0u;
    }
  }
  // ---- value scales in fp32, their largest magnitude per token
  float sv[2][NG], reach[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    reach[j] = 5.9604645e-8f;                    // 2^-24: a token whose values are all zero still counts in the sum
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&sc[j][(NG + g) >> 1]));
      sv[j][g] = (g & 1) ? two.y : two.x;
      reach[j] = fmaxf(reach[j], fabsf(sv[j][g]));
    }
  }
  float p[4];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = exp2_fast(fmaf(s[i], f.factor[i & 1], st.off[i & 1]));
    top = fmaxf(top, p[i] * reach[i >> 1]);
  }
  if (__any_sync(0xffffffffu, top > kQ4Limit)) {
    float next[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float most = fmaxf(fmaf(s[e], f.factor[e], log2_fast(reach[0])), fmaf(s[2 + e], f.factor[e], log2_fast(reach[1])));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
      next[e] = fminf(st.off[e], kQ4Top - most);
    }
    const bool far[2] = {fabsf(next[0]) >= kQ4Large, fabsf(next[1]) >= kQ4Large};       // also a column without a token yet
    if (__any_sync(0xffffffffu, far[0] || far[1] || st.off[0] == kQ4Far || st.off[1] == kQ4Far)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 old = st.place(e);
        float dot = fmaxf(s[e], s[2 + e]);
        dot = fmaxf(dot, __shfl_xor_sync(0xffffffffu, dot, 4));
        dot = fmaxf(dot, __shfl_xor_sync(0xffffffffu, dot, 8));
        dot = fmaxf(dot, __shfl_xor_sync(0xffffffffu, dot, 16));
        float2 now = make_float2(old.x != 0.f ? fmaxf(old.x, dot) : far[e] && dot > -INFINITY ? dot : 0.f, 0.f);
        float most = fmaxf(fmaf(s[e] - now.x, f.factor[e], log2_fast(reach[0])),
                           fmaf(s[2 + e] - now.x, f.factor[e], log2_fast(reach[1])));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
        const float same = fmaf(now.x - old.x, f.factor[e], old.y);           // what would leave every p as it is
        now.y = fminf(same, kQ4Top - most);
        st.rescale(e, exp2_fast(now.y - same));
        st.far[e] = now;
        st.off[e] = now.x != 0.f ? kQ4Far : now.y;
        p[e] = exp2_fast(fmaf(s[e] - now.x, f.factor[e], now.y));
        p[2 + e] = exp2_fast(fmaf(s[2 + e] - now.x, f.factor[e], now.y));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        st.rescale(e, exp2_fast(next[e] - st.off[e]));
        st.off[e] = next[e];
        p[e] = exp2_fast(fmaf(s[e], f.factor[e], next[e]));
        p[2 + e] = exp2_fast(fmaf(s[2 + e], f.factor[e], next[e]));
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) st.l[e] += p[e] + p[2 + e];
  // ---- V^T P^T
  uint32_t vw[T][2 * NG];
#pragma unroll
  for (int t = 0; t < T; ++t) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint4 u = *reinterpret_cast<const uint4*>(tiles + t * TILE + 256 * NG + i * 512 + lane * 16);
      vw[t][4 * i] = u.x; vw[t][4 * i + 1] = u.y; vw[t][4 * i + 2] = u.z; vw[t][4 * i + 3] = u.w;
    }
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint32_t b0 = transpose8(pack_f16x2(p[0] * sv[0][g], p[1] * sv[0][g]));
    const uint32_t b1 = transpose8(pack_f16x2(p[2] * sv[1][g], p[3] * sv[1][g]));
    const uint32_t eight = r == g ? 0x80088008u : 0u;                       // -8 * 2^-24 in row g
    mma_f16(st.z, eight, 0u, eight, 0u, b0, b1);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const uint32_t mine = T == 1 ? 0xffffffffu : (r >> 2) == t ? 0xffffffffu : 0u;   // the columns of this tile
      const uint32_t x0 = b0 & mine, x1 = b1 & mine;
      const uint32_t v0 = vw[t][g], v1 = vw[t][NG + g];
      const uint32_t w0 = __byte_perm(v0, 0u, 0x4341u), w1 = __byte_perm(v1, 0u, 0x4341u);     // the upper bytes
      mma_f16(st.o[g][0], v0 & 0x000f000fu, v0 & 0x00ff00ffu, v1 & 0x000f000fu, v1 & 0x00ff00ffu, x0, x1);
      mma_f16(st.o[g][1], w0 & 0x000f000fu, w0, w1 & 0x000f000fu, w1, x0, x1);
    }
  }
}

// Tiles of a row of the call; 0 for a row without tokens.
__device__ __forceinline__ int q4_len(const Q4DecodeArgs& a, int row) {
  const int len = min(a.lens[row], a.max_blocks * a.tiles * kQ4Tile);
  const int seq = a.seqs != nullptr ? a.seqs[row] : row;
  return seq < 0 || seq >= a.table_rows ? 0 : max(len, 0);
}
__device__ __forceinline__ int q4_count(int len) { return (len + kQ4Tile - 1) / kQ4Tile; }

// How the call's tiles are dealt out: unit = (row, slice of at most eight heads of a kv head), units in order, all tiles of all
// units in one line that is cut into equal ranges, one for each warp, so that lengths of any mixture keep every warp busy for
// the same time. A cut inside a unit of at most kQ4Whole tiles moves to its end: joining the parts of a short unit takes longer
// than a few more tiles. Every block finds the places of its warps by a sum over the rows' lengths. Lengths that change under
// the call, which are read more than once, make its results worthless but lead nowhere: rows, units and workers are held within
// their ranges here and where the parts are joined, and a cut within its unit.
struct Q4Plan {
  long long total;              // tiles of the call
  long long per;                // of a warp
  int units;                    // of a row
};

__device__ __forceinline__ Q4Plan q4_plan(const Q4DecodeArgs& a, int* rows, long long* before) {
  __shared__ long long sums[kQ4Warps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int each = (a.rows + kQ4Threads - 1) / kQ4Threads, first = threadIdx.x * each, last = min(a.rows, first + each);
  long long mine = 0;
  for (int row = first; row < last; ++row) mine += q4_count(q4_len(a, row));
  long long sum = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += up;
  }
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  long long ahead = sum - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kQ4Warps; ++w) {
    if (w < warp) ahead += sums[w];
    all += sums[w];
  }
  Q4Plan plan;
  plan.units = a.hkv * a.slices;
  plan.total = all * plan.units;
  const long long workers = (long long)gridDim.x * kQ4Warps, round = plan.total + workers - 1;
  plan.per = max((long long)kQ4MinTiles, round >> 32 ? round / workers : (long long)((uint32_t)round / (uint32_t)workers));
#pragma unroll
  for (int w = 0; w <= kQ4Warps; ++w) {           // the row that holds the first tile of warp w's range
    const long long at = ((long long)blockIdx.x * kQ4Warps + w) * plan.per;
    if (at < ahead * plan.units || at >= (ahead + mine) * plan.units) continue;
    long long b = ahead;
    int row = first;
    for (; row < last; ++row) {
      const int n = q4_count(q4_len(a, row));
      if (at < (b + n) * plan.units) break;
      b += n;
    }
    rows[w] = min(row, a.rows - 1);
    before[w] = b * plan.units;
  }
  __syncthreads();
  return plan;
}

// Four outputs of a head, at d, and its sum, of parts some of which have large scores: record(i) is the i-th one's.
template <typename R>
__device__ __forceinline__ void q4_join_large(float& sum, float4& acc, int parts, int d, R record, int hd) {
  float2 all = make_float2(0.f, kQ4None);
  sum = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i = 0; i < 2 * parts; ++i) {
    const float* x = record(i < parts ? i : i - parts);
    const float4 end = *reinterpret_cast<const float4*>(x + hd);
    const float2 place = end.x == kQ4Far ? make_float2(end.z, 0.f) : make_float2(0.f, end.x);
    if (i < parts) {
      all = q4_larger(all, place, end.w);
      continue;
    }
    const float4 o = *reinterpret_cast<const float4*>(x + d);
    const float by = q4_weight(place, all, end.w);
    sum += end.y * by;
    acc.x += o.x * by; acc.y += o.y * by; acc.z += o.z * by; acc.w += o.w * by;
  }
}

// A place in the line of tiles, relative to the warp's first.
struct Q4Cursor {
  int row, unit;                // unit within the row
  int begin, end;               // tiles of the unit
  int len;                      // tokens of the row
  __device__ __forceinline__ void next(const Q4DecodeArgs& a, int units) {
    begin = end;
    if (++unit == units) {
      unit = 0;
      do {
        ++row;
        len = row < a.rows ? q4_len(a, row) : kQ4Tile;
      } while (len == 0);
    }
    end = begin + q4_count(len);
  }
};

template <int NG, int T> __host__ __device__ constexpr int q4_stage() { return 576 * NG * T + 512 * NG / T; }
template <int NG, int T> __host__ __device__ constexpr int q4_stages() { return T == 1 ? 3 : 2; }
template <int NG, int T> __host__ __device__ constexpr int q4_smem() { return kQ4Warps * q4_stages<NG, T>() * q4_stage<NG, T>(); }

// Each warp goes its own way through its range: a ring of shared-memory stages, each T tiles and, at the start of a unit, the
// unit's query rows, filled by asynchronous copies that run ahead across units. A unit that lies within the range is finished
// from registers; parts of others go to `part` for the kernel below.
template <int NG, int T, bool BF16>
__global__ void __launch_bounds__(kQ4Threads, NG <= 2 ? 6 : NG <= 4 ? 4 : 2)
paged_decode_q4_kernel(const __grid_constant__ Q4DecodeArgs a) {
  constexpr int HD = NG * 32, TILE = 576 * NG, STAGE = q4_stage<NG, T>(), STAGES = q4_stages<NG, T>(), REC = HD + 4;
  constexpr int COLUMNS = 8 / T;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int plan_rows[kQ4Warps + 1];
  __shared__ long long plan_before[kQ4Warps + 1];
  __shared__ float2 far[kQ4Threads][2];
  wait_for_previous();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int group = a.hq / a.hkv;
  const int worker = blockIdx.x * kQ4Warps + warp;
  const Q4Plan plan = q4_plan(a, plan_rows, plan_before);
  // ---- this warp's range
  Q4Cursor now;
  long long start;
  int count;
  {
    long long at[2];
#pragma unroll
    for (int i = 1; i >= 0; --i) {
      at[i] = min(plan.total, (worker + i) * plan.per);
      if (at[i] == plan.total) continue;
      const int row = plan_rows[warp + i], len = q4_len(a, row), n = q4_count(len);
      const uint32_t into = (uint32_t)(at[i] - plan_before[warp + i]);
      const uint32_t unit = min(into / (uint32_t)max(n, 1), (uint32_t)plan.units - 1);
      const int off = (int)min(into - unit * n, (uint32_t)n);
      now.row = row;
      now.unit = unit;
      now.len = len;
      now.begin = -off;
      now.end = now.begin + n;
      if (off > 0 && n <= kQ4Whole) {
        at[i] += n - off;
        now.end = 0;
        now.next(a, plan.units);
      }
    }
    start = at[0];
    count = (int)(at[1] - at[0]);
  }
  int4 owner = make_int4(-1, 0, 0, 0);
  if (count > 0) {
    uint8_t* ring = smem + warp * STAGES * STAGE;
    const uint32_t to0 = smem_u32(ring) + lane * 16;
    const uint8_t* from0 = a.pool + lane * 16;
    // Tiles to come, 32 at a time: lane i looks up the place of the i-th (its number among the pool's tiles; -1: not in the
    // pool, or behind the range), all in one unit.
    Q4Cursor ahead = now;
    int fetched = 0, list = -1, at = 0, filled = 0;        // tiles listed so far, this lane's, next one of the list, its length
    bool entered = false;                                  // the unit that `ahead` is in has been begun
    uint32_t stage_in = 0, missing = 0;                    // bits: tiles that are not there, the last one issued lowest
    auto refill = [&]() {
      at = 0;
      filled = 32;
      list = -1;
      if (fetched >= count) return;
      if (fetched == ahead.end) {
        ahead.next(a, plan.units);
        entered = false;
      }
      const int kvh = a.slices == 1 ? ahead.unit : ahead.unit / a.slices;
      const int row = min(ahead.row, a.rows - 1);
      if (!entered) {                                      // the unit's query rows travel with its first tile
        const int g0 = (ahead.unit - kvh * a.slices) * 8, pieces = min(COLUMNS, group - g0) * (HD / 8);
        const uint16_t* q = a.q + (size_t)row * a.q_stride + (size_t)(kvh * group + g0) * HD;
        for (int i = lane; i < pieces; i += 32) copy16(to0 + stage_in + T * TILE + (i - lane) * 16, q + i * 8);
        entered = true;
      }
      filled = min(32, min(ahead.end, count) - fetched);
      if (lane < filled) {
        const int seq = a.seqs != nullptr ? max(0, min(a.seqs[row], a.table_rows - 1)) : row;
        const int t = fetched + lane - ahead.begin, page = min(a.tiles == 1 ? t : t / a.tiles, a.max_blocks - 1);
        const int block = a.block_table[(size_t)seq * a.max_blocks + page];
        if ((uint32_t)block < (uint32_t)a.num_blocks)
          list = (block * a.hkv + kvh) * a.tiles + min(t - page * a.tiles, a.tiles - 1);
      }
      fetched += filled;
    };
    auto issue = [&]() {
      if (at >= filled) refill();
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int tile = __shfl_sync(0xffffffffu, list, at + t);
        missing = missing * 2 + (tile < 0);
        copy_tile<NG>(to0 + stage_in + t * TILE, from0 + (size_t)(uint32_t)max(tile, 0) * TILE, tile >= 0);
      }
      at += T;
      asm volatile("cp.async.commit_group;" ::: "memory");
      stage_in = stage_in == (STAGES - 1) * STAGE ? 0 : stage_in + STAGE;
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) issue();

    Q4Query<NG, T> f;
    Q4State<NG> st;
    st.far = far[threadIdx.x];
    int mine = 0;
    const uint8_t* tiles = ring;
    for (;;) {
      const int kvh = a.slices == 1 ? now.unit : now.unit / a.slices, g0 = (now.unit - kvh * a.slices) * 8;
      const int heads = min(COLUMNS, group - g0), head0 = kvh * group + g0;
      st.clear();
      const int stop = min(now.end, count);
      int live = now.len - (mine - now.begin) * kQ4Tile;
      for (bool first = true; mine < stop; mine += T, live -= T * kQ4Tile, first = false) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                            // all lanes' pieces have landed; the previous stage has been read
        const uint32_t gone = missing >> ((STAGES - 2) * T) & ((1u << T) - 1u);
        if (first) q4_load_query<NG, T, BF16>(f, tiles + T * TILE, heads, a.scale, a.scale_exp);
        issue();
        if (NG <= 4 && live >= T * kQ4Tile && gone == 0u) q4_pass<NG, T, true>(st, f, tiles, live, gone);
        else q4_pass<NG, T, false>(st, f, tiles, live, gone);
        tiles = tiles == ring + (STAGES - 1) * STAGE ? ring : tiles + STAGE;
      }
      mine = stop;
      // ---- the unit, or the warp's part of it
      const bool begins = now.begin >= 0, ends = now.end <= count, whole = begins && ends;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], off);
      }
      if (T == 2) st.fold(f.factor);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 2 * c + e;
        // slot 0: the unit began before this range; slot 1: it goes on after it
        float* rec = a.part + (((size_t)worker * 2 + (begins ? 1 : 0)) * a.heads + h) * REC;
        const float4 end = st.end(e, f.factor[e]);
        const float by = !whole ? 16777216.f : st.l[e] == 0.f ? 0.f : 16777216.f / st.l[e];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float z = __shfl_sync(0xffffffffu, st.z[e], 4 * g + c);
          const float4 o = make_float4((st.o[g][0][e] + z) * by, fmaf(st.o[g][0][2 + e] - st.o[g][0][e], 0.0625f, z) * by,
                                       (st.o[g][1][e] + z) * by, fmaf(st.o[g][1][2 + e] - st.o[g][1][e], 0.0625f, z) * by);
          if (h >= heads || now.row >= a.rows) continue;
          uint16_t* to = a.out + (size_t)now.row * a.out_stride + (size_t)(head0 + h) * HD + 32 * g + 4 * r;
          if (whole) q4_store4<BF16>(to, o.x, o.y, o.z, o.w);
          else *reinterpret_cast<float4*>(rec + 32 * g + 4 * r) = o;
        }
        if (!whole && h < heads && r == 0) *reinterpret_cast<float4*>(rec + HD) = end;
      }
      if (begins) {
        owner = whole ? make_int4(-1, 0, 0, 0) : make_int4(now.row, now.unit, worker, (int)((start + now.end - 1) / plan.per));
        if (a.by_unit && lane == 0 && now.row < a.rows) a.owner[(size_t)now.row * plan.units + now.unit] = owner;
      }
      if (now.end >= count) break;
      now.next(a, plan.units);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  if (!a.by_unit && lane == 0) a.owner[worker] = owner;
  // rows without tokens
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (q4_len(a, row) > 0) continue;
    for (int i = threadIdx.x * 4; i < a.hq * HD; i += kQ4Threads * 4)
      q4_store4<BF16>(a.out + (size_t)row * a.out_stride + i, 0.f, 0.f, 0.f, 0.f);
    if (a.by_unit)
      for (int u = threadIdx.x; u < plan.units; u += kQ4Threads) a.owner[(size_t)row * plan.units + u] = make_int4(-1, 0, 0, 0);
  }
}

// Shared memory of one of its warps, besides Q4State::far: the ring, and once that is done with, a record of each column.
template <int NG, int T> __host__ __device__ constexpr int q4_each() {
  constexpr int ring = q4_stages<NG, T>() * q4_stage<NG, T>(), records = 8 * (NG * 32 + 4) * 4;
  return ring > records ? ring : records;
}
constexpr int kQ4FarBytes = 32 * 2 * sizeof(float2);

// A block for each unit, whose warps take turns with its tiles and meet in shared memory: one launch, nothing to plan, two
// dependent loads before the first tile. For tables so narrow that the longest unit keeps its warps busy only shortly.
template <int NG, int T, bool BF16>
__global__ void __launch_bounds__(NG <= 4 ? 512 : 256) paged_decode_q4_unit_kernel(const __grid_constant__ Q4DecodeArgs a) {
  constexpr int HD = NG * 32, TILE = 576 * NG, STAGE = q4_stage<NG, T>(), STAGES = q4_stages<NG, T>(), REC = HD + 4;
  constexpr int COLUMNS = 8 / T;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warps = blockDim.x >> 5, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int units = a.hkv * a.slices, row = blockIdx.x / units, unit = blockIdx.x - row * units, group = a.hq / a.hkv;
  const int kvh = a.slices == 1 ? unit : unit / a.slices, g0 = (unit - kvh * a.slices) * 8;
  const int heads = min(COLUMNS, group - g0), head0 = kvh * group + g0;
  wait_for_previous();
  const int len = q4_len(a, row), n = q4_count(len), passes = (n + T - 1) / T;
  // passes warp, warp + warps, ... are this warp's; lane i looks up the place of its i-th tile from `listed` on
  uint8_t* ring = smem + warp * STAGES * STAGE;
  const uint32_t to0 = smem_u32(ring) + lane * 16;
  const uint8_t* from0 = a.pool + lane * 16;
  const int seq = a.seqs != nullptr ? max(0, min(a.seqs[row], a.table_rows - 1)) : row;
  const int* pages = a.block_table + (size_t)seq * a.max_blocks;
  int listed = 0, list = -1;
  auto refill = [&]() {
    const int i = listed + lane, t = (warp + i / T * warps) * T + i % T;
    const int page = a.tiles == 1 ? t : t / a.tiles;
    // read whether the row has the tile or not: the first of these does not wait for the row's length
    const int block = a.max_blocks > 0 ? pages[min(page, a.max_blocks - 1)] : -1;
    list = t < n && (uint32_t)block < (uint32_t)a.num_blocks ? (block * a.hkv + kvh) * a.tiles + (t - page * a.tiles) : -1;
    listed += 32;
  };
  int at = 0;
  uint32_t stage_in = 0, missing = 0;
  auto issue = [&]() {
    if (at == listed) refill();
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int tile = __shfl_sync(0xffffffffu, list, (at + t) & 31);
      missing = missing * 2 + (tile < 0);
      copy_tile<NG>(to0 + stage_in + t * TILE, from0 + (size_t)(uint32_t)max(tile, 0) * TILE, tile >= 0);
    }
    at += T;
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_in = stage_in == (STAGES - 1) * STAGE ? 0 : stage_in + STAGE;
  };
  if (warp < passes) {
    const uint16_t* q = a.q + (size_t)row * a.q_stride + (size_t)head0 * HD;
    for (int i = lane; i < heads * (HD / 8); i += 32) copy16(to0 + T * TILE + (i - lane) * 16, q + i * 8);
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) issue();
  }
  Q4Query<NG, T> f;
  Q4State<NG> st;
  st.far = reinterpret_cast<float2*>(smem + warps * q4_each<NG, T>()) + 2 * threadIdx.x;
  st.clear();
  const uint8_t* tiles = ring;
  for (int pass = warp; pass < passes; pass += warps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                // all lanes' pieces have landed; the previous stage has been read
    const uint32_t gone = missing >> ((STAGES - 2) * T) & ((1u << T) - 1u);
    if (pass == warp) q4_load_query<NG, T, BF16>(f, tiles + T * TILE, heads, a.scale, a.scale_exp);
    issue();
    const int live = len - pass * T * kQ4Tile;
    if (NG <= 4 && live >= T * kQ4Tile && gone == 0u) q4_pass<NG, T, true>(st, f, tiles, live, gone);
    else q4_pass<NG, T, false>(st, f, tiles, live, gone);
    tiles = tiles == ring + (STAGES - 1) * STAGE ? ring : tiles + STAGE;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], off);
  }
  __syncthreads();                               // the ring becomes the meeting place: [warp][column] records
  float* records = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float* rec = records + (warp * 8 + 2 * c + e) * REC;
    const float4 end = st.end(e, f.factor[e]);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float z = __shfl_sync(0xffffffffu, st.z[e], 4 * g + c);
      *reinterpret_cast<float4*>(rec + 32 * g + 4 * r) =
          make_float4(st.o[g][0][e] + z, fmaf(st.o[g][0][2 + e] - st.o[g][0][e], 0.0625f, z), st.o[g][1][e] + z, fmaf(st.o[g][1][2 + e] - st.o[g][1][e], 0.0625f, z));
    }
    if (r == 0) *reinterpret_cast<float4*>(rec + HD) = end;
  }
  __syncthreads();
  const int parts = min(warps, passes) * T;      // of a head: column h of each warp, and h + 4 with T = 2
  for (int i = threadIdx.x; i < heads * (HD / 4); i += blockDim.x) {
    const int h = i / (HD / 4), d = (i - h * (HD / 4)) * 4;
    const float* rec = records + h * REC;
    float off = kQ4None, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    bool large = false;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      off = fminf(off, rec[p * COLUMNS * REC + HD]);
      large |= rec[p * COLUMNS * REC + HD] == kQ4Far;
    }
    if (large) {
      q4_join_large(sum, acc, parts, d, [&](int p) { return rec + p * COLUMNS * REC; }, HD);
    } else {
#pragma unroll 4
      for (int p = 0; p < parts; ++p) {
        const float* x = rec + p * COLUMNS * REC;
        const float by = exp2_fast(off - x[HD]);
        const float4 o = *reinterpret_cast<const float4*>(x + d);
        sum += x[HD + 1] * by;
        acc.x += o.x * by; acc.y += o.y * by; acc.z += o.z * by; acc.w += o.w * by;
      }
    }
    const float by = sum == 0.f ? 0.f : 16777216.f / sum;
    uint16_t* to = a.out + (size_t)row * a.out_stride + (size_t)(head0 + h) * HD + d;
    q4_store4<BF16>(to, acc.x * by, acc.y * by, acc.z * by, acc.w * by);
  }
}

// Joins the parts of units that several warps share: slot 1 of the warp that began it, slot 0 of the others. A task is a head of
// an entry of `owner`. SPREAD: few long units; a block does one task, its groups of HD / 4 threads take turns with the records and
// meet in shared memory. Otherwise each group of threads does a task by itself.
constexpr int kQ4MergeThreads = 256;

template <int NG, bool BF16, bool SPREAD>
__global__ void __launch_bounds__(kQ4MergeThreads)
paged_decode_q4_merge_kernel(const __grid_constant__ Q4DecodeArgs a, long long tasks) {
  constexpr int HD = NG * 32, REC = HD + 4, LANES = HD / 4, SETS = kQ4MergeThreads / LANES, DEPTH = 8;
  __shared__ __align__(16) float sm_o[SPREAD ? SETS : 1][HD];
  __shared__ float sm_off[SETS], sm_l[SETS];
  const int set = threadIdx.x / LANES, d = (threadIdx.x - set * LANES) * 4, group = a.hq / a.hkv;
  const long long task = SPREAD ? blockIdx.x : (long long)blockIdx.x * SETS + set;
  wait_for_previous();
  if (task >= tasks || (!SPREAD && set >= SETS)) return;
  const long long entry = task / a.heads;
  const int h = (int)(task - entry * a.heads);
  const int4 owner = a.owner[entry];
  // -1: nothing to join; what else is out of range only lengths that changed under the call leave here
  if ((uint32_t)owner.x >= (uint32_t)a.rows || (uint32_t)owner.y >= (uint32_t)(a.hkv * a.slices) || owner.z < 0 ||
      owner.w >= a.workers)
    return;
  const int kvh = owner.y / a.slices, g0 = (owner.y - kvh * a.slices) * 8;
  if (h >= group - g0) return;
  float off = kQ4None, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  bool large = false;
  constexpr int STEP = SPREAD ? SETS : 1;
  auto record = [&](int w) { return a.part + (((size_t)w * 2 + (w == owner.z ? 1 : 0)) * a.heads + h) * REC; };
  for (int w0 = owner.z + (SPREAD ? set : 0); w0 <= owner.w && set < SETS; w0 += DEPTH * STEP) {
    float2 x[DEPTH];
    float4 o[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {            // all on the way before the first is used
      const int w = w0 + i * STEP;
      x[i] = make_float2(kQ4None, 0.f);
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (w > owner.w) continue;
      const float* rec = record(w);
      x[i] = *reinterpret_cast<const float2*>(rec + HD);
      o[i] = *reinterpret_cast<const float4*>(rec + d);
    }
    float next = off;
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      next = fminf(next, x[i].x);
      large |= x[i].x == kQ4Far;
    }
    const float by = exp2_fast(next - off);
    sum *= by; acc.x *= by; acc.y *= by; acc.z *= by; acc.w *= by;
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      const float y = exp2_fast(next - x[i].x);
      sum += x[i].y * y;
      acc.x += o[i].x * y; acc.y += o[i].y * y; acc.z += o[i].z * y; acc.w += o[i].w * y;
    }
    off = next;
  }
  if (SPREAD) {
    if (set < SETS) {
      *reinterpret_cast<float4*>(&sm_o[set][d]) = acc;
      if (d == 0) { sm_off[set] = off; sm_l[set] = sum; }
    }
    large = __syncthreads_or(large);
    if (set > 0) return;
    float all = kQ4None;
#pragma unroll
    for (int s = 0; s < SETS; ++s) all = fminf(all, sm_off[s]);
    sum = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const float x = exp2_fast(all - sm_off[s]);
      const float4 v = *reinterpret_cast<const float4*>(&sm_o[s][d]);
      sum += sm_l[s] * x;
      acc.x += v.x * x; acc.y += v.y * x; acc.z += v.z * x; acc.w += v.w * x;
    }
  }
  if (large) q4_join_large(sum, acc, owner.w - owner.z + 1, d, [&](int i) { return record(owner.z + i); }, HD);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  q4_store4<BF16>(a.out + (size_t)owner.x * a.out_stride + (size_t)(kvh * group + g0 + h) * HD + d, acc.x * inv, acc.y * inv,
                  acc.z * inv, acc.w * inv);
}

// Blocks of the attention kernel that the GPU holds at a time: the most of a call.
template <int NG, int T, bool BF16>
static int q4_blocks() {
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  int& n = known[dev];
  if (n == 0) {
    int per_sm = 0;
    auto k = paged_decode_q4_kernel<NG, T, BF16>;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, q4_smem<NG, T>()) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, kQ4Threads, q4_smem<NG, T>()) != cudaSuccess || per_sm < 1)
      return -1;
    n = per_sm * num_sms();
  }
  return n;
}

// Warps of a block of the kernel for whole units; 0: the call goes to the kernel for ranges. Enough of them to fill the GPU with
// ten warps to an SM, no more than two tiles each need, and so many that none has more than 32 tiles, for a long row among
// short ones is its block's alone. Ranges cost some 10 us more, of which a part of a few tiles is too much to wait for them where
// the units are few: what a warp has here beyond an even share of all tiles may be ten tiles of 128 elements a head. With
// 128-element heads, this kernel and ranges, us: 512 rows of 768 tokens on 2 kv heads 28.4, 38.7; of 1536 46.3, 59.3; 8 of 4000 on
// 32 30.9, 35.5; 64 of 8000 on 2 33.3, 44.0; 8 of 4000 on 8 17.9, 19.8; but 4 of 4000 on 8 17.6, 15.4; 16 of 8000 on 2 32.4, 20.7;
// 4 of 30000 on 8 92.2, 35.8; 48 of up to 10000 on 8 67.8, 65.2. 64 rows of 4000 on 1 of 256: 37.2, 28.1.
// The rule knows the table's width and not the lengths, which are on the device: in tables much wider than their rows most warps of
// a block have nothing. 512 rows of 100 tokens on 2 kv heads: 10.0 us in a table of 112 tokens, 10.2 in 1024, 12.9 in 2048, 19.5 in
// 4096, 32 in 8192; of 768 tokens 28.7 in 768, 28.1 in 1536, 53 in 8192; one row of 8000 among 255 of 100 32.1 (24.9 by ranges).
static int q4_unit_warps(int hd, long long units, long long tiles) {
  const int most = hd <= 128 ? 16 : 8;
  int warps = 1;
  while (warps < most && ((units * warps < 10LL * num_sms() && tiles > 2 * warps) || tiles > 32 * warps)) warps *= 2;
  const long long held = (hd <= 64 ? 24LL : hd <= 128 ? 16LL : 8LL) * num_sms();       // warps that the GPU holds
  const long long beyond = tiles / warps - units * tiles / held;
  return tiles <= 32 * warps && beyond * hd <= 10 * 128 && units <= 0x7fffffffLL ? warps : 0;
}

template <int NG, int T, bool BF16>
static int launch_q4_units(const Q4DecodeArgs& a, int warps, long long units, cudaStream_t st) {
  auto k = paged_decode_q4_unit_kernel<NG, T, BF16>;
  constexpr int each = q4_each<NG, T>() + kQ4FarBytes;
  static int ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (NG <= 4 ? 16 : 8) * each) != cudaSuccess)
      return -5;
    ready[dev] = 1;
  }
  return launch_behind("paged_decode_q4", k, (unsigned)units, warps * 32, warps * each, st, a);
}

template <int NG, int T, bool BF16>
static int launch_q4_decode(Q4DecodeArgs& a, int blocks, cudaStream_t st) {
  if (blocks > q4_blocks<NG, T, BF16>()) return -5;
  const long long units = (long long)a.rows * a.hkv * a.slices, workers = (long long)blocks * kQ4Warps;
  a.workers = (int)workers;
  a.by_unit = units <= workers;                  // an entry for each unit or each warp, whichever are fewer
  const int rc = launch_behind("paged_decode_q4", paged_decode_q4_kernel<NG, T, BF16>, blocks, kQ4Threads, q4_smem<NG, T>(), st,
                               a);
  if (rc != 0) return rc;
  const bool spread = units * 8 < workers;       // more than eight parts to a unit
  const long long tasks = (a.by_unit ? units : workers) * a.heads;
  constexpr int SETS = kQ4MergeThreads / (NG * 8);
  const unsigned grid = (unsigned)(spread ? tasks : (tasks + SETS - 1) / SETS);
  auto merge = spread ? paged_decode_q4_merge_kernel<NG, BF16, true> : paged_decode_q4_merge_kernel<NG, BF16, false>;
  return launch_behind("paged_decode_q4_merge", merge, grid, kQ4MergeThreads, 0, st, a, tasks);
}

// What a call needs of a variant: blocks of the kernel for ranges that fit the GPU (RUN false), or the call itself. T = 2 where
// at most four query heads share a kv head, whose passes over one tile would leave half of the columns idle: 4 rows of 100000
// tokens, 32 heads on 8, took 112 us with T = 1 and 107 with T = 2 in the same state of the rest.
template <bool RUN>
static int q4_variant(int hd, int per, int dtype, Q4DecodeArgs* a, int blocks, int warps, cudaStream_t st) {
#define ICB_Q4(NG_, T_, BF_) \
  if (hd == NG_ * 32 && (per > 4 ? 1 : 2) == T_ && dtype == (BF_ ? kBF16 : kF16)) { \
    if (RUN && warps > 0) return launch_q4_units<NG_, T_, BF_>(*a, warps, (long long)a->rows * a->hkv * a->slices, st); \
    if (RUN) return launch_q4_decode<NG_, T_, BF_>(*a, blocks, st); \
    return q4_blocks<NG_, T_, BF_>(); \
  }
#define ICB_Q4_TYPES(NG_) ICB_Q4(NG_, 1, true) ICB_Q4(NG_, 2, true) ICB_Q4(NG_, 1, false) ICB_Q4(NG_, 2, false)
  ICB_Q4_TYPES(2) ICB_Q4_TYPES(4) ICB_Q4_TYPES(6) ICB_Q4_TYPES(8)
#undef ICB_Q4_TYPES
#undef ICB_Q4
  return -3;
}

}  // namespace icb

using namespace icb;

// How icb_paged_decode_q4 is to run a call of `units` = rows * hkv * ceil(hq / hkv / 8) whose table rows hold `tiles` times 16
// tokens: positive, the `warps` of a block for each unit; negative, minus the `blocks` that share the tiles. 0: not covered.
ICB_API int icb_paged_decode_q4_plan(int hd, int per, int dtype, long long units, long long tiles) {
  const int fit = q4_variant<false>(hd, per, dtype, nullptr, 0, 0, nullptr);
  if (fit < 1) return 0;
  const int warps = q4_unit_warps(hd, units, tiles);
  if (warps > 0) return warps;
  const long long need = (units * tiles + kQ4Warps * kQ4MinTiles - 1) / (kQ4Warps * kQ4MinTiles);
  return -(int)(need < 1 ? 1 : need < fit ? need : fit);
}

// The arguments of icb_paged_decode_q4 come as one record: a caller through ctypes packs it in 0.7 us, where 22 arguments by
// themselves took 3.4 us of the 9 that a short call takes on the host.
//   q: [rows, hq * hd] 16-bit rows of pitch q_stride (16-byte aligned); pool: num_blocks pages of [hkv][tiles] tiles; row i
//   attends over the first lens[i] tokens of table row seqs[i] (null: i). out: [rows, out_stride], same type. hd 64, 128, 192
//   or 256. plan: as icb_paged_decode_q4_plan gives it; where it is negative, scratch has blocks * 4 * (4 + 2 * min(8, hq / hkv)
//   * (hd + 4)) floats, 16-byte aligned.
struct Q4DecodeCall {
  const uint16_t* q;
  long long q_stride;
  const uint8_t* pool;
  const int *block_table, *seqs, *lens;
  uint16_t* out;
  long long out_stride;
  float* scratch;
  long long rows, hq, hkv, hd, tiles, max_blocks, table_rows, num_blocks, plan;
  double scale;
  long long dtype;
};

ICB_API int icb_paged_decode_q4(const void* record, void* stream) {
  Q4DecodeCall c;
  memcpy(&c, record, sizeof(c));
  if (c.rows <= 0) return 0;
  if (c.hkv < 1 || c.hq < 1 || c.hq % c.hkv || c.tiles < 1 || c.q_stride % 8) return -2;
  if (c.plan == 0 || c.plan > (c.hd <= 128 ? 16 : 8)) return -2;
  const long long per = c.hq / c.hkv, slices = (per + 7) / 8, blocks = c.plan < 0 ? -c.plan : 0;
  // the numbers of a pool's tiles and of a row's tiles in all units are 32-bit
  if (c.max_blocks * c.tiles * c.hkv * slices > 0x7fffffffLL || c.max_blocks * c.tiles > 0x7ffffffLL ||
      c.num_blocks * c.hkv * c.tiles > 0x7fffffffLL || c.rows * c.hkv * slices > 0x7fffffffLL || c.hq > 0x7fffffffLL ||
      c.table_rows > 0x7fffffffLL || blocks > 0x7fffffffLL)
    return -2;
  Q4DecodeArgs a{c.q, c.q_stride, c.pool, c.block_table, c.seqs, c.lens, c.out, c.out_stride,
                 reinterpret_cast<int4*>(c.scratch), 0, c.scratch + (size_t)blocks * kQ4Warps * 4,
                 (int)c.rows, (int)c.hq, (int)c.hkv, (int)slices, (int)(per < 8 ? per : 8), (int)c.tiles, (int)c.max_blocks,
                 (int)c.table_rows, (int)c.num_blocks, 0, 0.f, 0};
  a.scale = (float)frexp(c.scale, &a.scale_exp) * kLog2e;
  return q4_variant<true>((int)c.hd, (int)per, (int)c.dtype, &a, (int)blocks, c.plan > 0 ? (int)c.plan : 0,
                          reinterpret_cast<cudaStream_t>(stream));
}
