// Attention of single query rows over the 4-bit paged cache (format: q4.cuh) on sm_100a.
//
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q . k_t),  k_td = sk_tg (n_td - 8),  v_td = sv_tg (m_td - 8)
//
// Up to eight query heads of a kv head's group are the N dimension of mma.sync.m16n8k16 (fp16, fp32 sums), 16 tokens the M
// dimension of K Q^T and 16 elements that of V^T P^T: every row of the matrix instructions is used.
//   * A code needs no conversion: four bits at the bottom of an fp16 are the number n 2^-24, exact in the matrix
//     instruction, so a word & 0x000f000f is two operands, & 0x00f000f0 two more that are 16 n 2^-24. The factor 16 is taken
//     out of the query elements beforehand and out of the output rows at the end; shifted by 8 the word gives the other four.
//   * q . (n - 8) = q . n - 8 sum q: the second part is a product of the key scales with a constant of the query, one matrix
//     instruction for all groups (the constant as fp16 plus what fp16 leaves of it, 22 bits). On the value side another one,
//     whose constant operand has -8 in row g, sums -8 p_t sv_tg from the same rounded products.
//   * The scale of a group multiplies a finished dot product (keys) or the probability before it is rounded to fp16 (values).
//   * Queries are scaled per head by a power of two to [2^14, 2^15) so that bf16 fits fp16: an element loses bits only below
//     2^-24 of the head's largest.
//   * p_t sv_tg is rounded to fp16 too. Its range is held by the maximum that the softmax subtracts: it runs over
//     log2 p_t + log2 max_g |sv_tg| instead of log2 p_t, so that the largest product is 2^12 to 2^15, whatever the values'
//     magnitude. Relative error 2^-11 down to 2^-26 of the largest contribution; sums, maxima and p itself stay in fp32.
// Tokens outside the sequence get probability and value scale zero by selection, so nothing stale in a page (NaN scales
// included) reaches a result. A page number outside the pool counts as a page outside the sequence.
#include "host_common.h"
#include "ptx.cuh"
#include "q4.cuh"

namespace icb {

constexpr int kQ4Warps = 4;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4MinTiles = 2;                  // least tiles of a warp
constexpr int kQ4Whole = 8;                     // units of at most so many tiles are not divided among warps
constexpr float kQ4Top = 12.f;                  // log2 of the largest fp16 probability times scale right after a new maximum
constexpr float kQ4Limit = 32768.f;             // and what it may grow to before the maximum is taken again: fp16 holds it
constexpr float kQ4None = -1e30f;               // maximum of no tokens
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
  int4* owner;                  // [workers]: {row, unit, last worker} of a unit that begins in a worker's range and goes on
  float* part;                  // [workers][2][slice heads] records of HD + 4 floats: outputs, maximum, sum
  int rows, hq, hkv, slices, heads, tiles, max_blocks, table_rows, num_blocks;   // heads: of a slice, at most eight
  float scale;                  // score factor times log2(e)
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

// The query operand of up to eight heads, resident in registers.
template <int NG>
struct Q4Query {
  uint32_t b[NG][4];            // B fragments of the two matrix instructions of a group
  uint32_t start[NG > 4 ? 2 : 1];   // B fragment of -8 * sum of a group's query elements: fp16 and what it leaves
  float factor[2], factor8[2];  // from the dot products, and from the sums of `start`, to the base-2 score; heads 2c, 2c + 1
};

template <int NG, bool BF16>
__device__ __forceinline__ void q4_load_query(Q4Query<NG>& f, const uint8_t* q, int heads, float scale) {
  constexpr int HD = NG * 32;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  float x[NG][8];
  float top = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (r < heads) u = *reinterpret_cast<const uint4*>(q + (r * HD + g * 32 + c * 8) * 2);
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
  const int e = min(max((__float_as_int(top) >> 23) - 127, -100), 116);
  const float up = __int_as_float((127 + 14 - e) << 23), up16 = up * 0.0625f;
  const float back = __int_as_float((127 + 10 + e) << 23) * scale;           // 2^24 / up
  float start[NG > 4 ? 2 : 1] = {};
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
    if ((g & 3) == c) start[g >> 2] = sum;                                   // k slots 2c, 2c + 1 belong to group c (and c + 4)
  }
#pragma unroll
  for (int i = 0; i < (NG > 4 ? 2 : 1); ++i) {
    const float x = start[i] * (-8.f / 256.f);                               // |sum| <= 2^20: at most 2^15
    const __half hi = __float2half_rn(x);
    const __half2 both = __halves2half2(hi, __float2half_rn(x - __half2float(hi)));
    f.start[i] = *reinterpret_cast<const uint32_t*>(&both);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    f.factor[e] = __shfl_sync(0xffffffffu, back, 8 * c + 4 * e);             // head 2c + e: lanes 4 (2c + e) ..
    f.factor8[e] = f.factor[e] * (256.f / 16777216.f);
  }
}

// Running state of a warp: this lane's part of eight heads.
template <int NG>
struct Q4State {
  float o[NG][2][4];            // V^T P^T: elements 32 g + 4 r + 2 m + (reg >> 1), heads 2c + (reg & 1); odd elements times 16
  float z[4];                   // row g: -8 * sum of the rounded p * value scale of group g, in the units of o (even elements)
  float m[2], l[2];             // what is subtracted for heads 2c, 2c + 1 (equal in all lanes r), sum of this lane's p
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[g][0][i] = o[g][1][i] = 0.f;
    }
    z[0] = z[1] = z[2] = z[3] = 0.f;
    m[0] = m[1] = kQ4None;
    l[0] = l[1] = 0.f;
  }
};

// One tile of 16 tokens in shared memory; `live` of them belong to the sequence (16 or more: all).
template <int NG>
__device__ __forceinline__ void q4_tile(Q4State<NG>& st, const Q4Query<NG>& f, const uint8_t* tile, int live) {
  constexpr int NP = NG / 2;                     // 16-byte pieces per lane of the keys, and of the values
  const int lane = threadIdx.x & 31, r = lane >> 2;
  // scales of tokens r and r + 8: NG fp16 of the keys, NG of the values
  uint32_t sc[2][NG];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint8_t* at = tile + 512 * NG + (r + 8 * j) * 4 * NG;
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
  // ---- scores of tokens r, r + 8 and heads 2c, 2c + 1: s[j][e]
  float s[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  float base8[4];                                // sum over the groups of key scale * start: rows are tokens again
  {
    const uint32_t pick = 0x1010u + 0x2222u * (NG == 2 ? lane & 1 : lane & 3);       // scale of group c, twice
    const uint32_t a0 = __byte_perm(sc[0][0], sc[0][NG == 2 ? 0 : 1], pick), a1 = __byte_perm(sc[1][0], sc[1][NG == 2 ? 0 : 1], pick);
    if (NG <= 4) {
      mma_f16_first(base8, a0, a1, 0u, 0u, f.start[0], 0u);
    } else {
      const uint32_t pick2 = 0x1010u + 0x2222u * (NG == 6 ? lane & 1 : lane & 3);    // and of group c + 4
      constexpr int K2 = NG > 4 ? 2 : 0, K3 = NG == 8 ? 3 : K2;
      mma_f16_first(base8, a0, a1, __byte_perm(sc[0][K2], sc[0][K3], pick2), __byte_perm(sc[1][K2], sc[1][K3], pick2), f.start[0],
              f.start[NG > 4 ? 1 : 0]);
    }
  }
  {
    uint32_t kw[2 * NG];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint4 u = *reinterpret_cast<const uint4*>(tile + p * 512 + lane * 16);
      kw[4 * p] = u.x; kw[4 * p + 1] = u.y; kw[4 * p + 2] = u.z; kw[4 * p + 3] = u.w;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float d[4];
      const uint32_t a = kw[g], b = kw[NG + g];
      mma_f16_first(d, a & 0x000f000fu, b & 0x000f000fu, a & 0x00f000f0u, b & 0x00f000f0u, f.b[g][0], f.b[g][1]);
      const uint32_t a8 = a >> 8, b8 = b >> 8;
      mma_f16(d, a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u, f.b[g][2], f.b[g][3]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&sc[j][g >> 1]));
        const float ks = (g & 1) ? two.y : two.x;
        s[j][0] = fmaf(ks, d[2 * j], s[j][0]);
        s[j][1] = fmaf(ks, d[2 * j + 1], s[j][1]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j][e] = fmaf(base8[2 * j + e], f.factor8[e], s[j][e] * f.factor[e]);
  }
  if (live < kQ4Tile) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (r + 8 * j < live) continue;
      s[j][0] = s[j][1] = -INFINITY;
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
  float p[2][2];
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      p[j][e] = exp2_fast(s[j][e] - st.m[e]);
      top = fmaxf(top, p[j][e] * reach[j]);
    }
  }
  if (__any_sync(0xffffffffu, top > kQ4Limit)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float most = fmaxf(s[0][e] + log2_fast(reach[0]), s[1][e] + log2_fast(reach[1]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
      const float next = fmaxf(st.m[e], most - kQ4Top);
      const float corr = exp2_fast(st.m[e] - next);
      st.m[e] = next;
      st.l[e] *= corr;
      st.z[e] *= corr;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int t = 0; t < 2; ++t) { st.o[g][t][e] *= corr; st.o[g][t][2 + e] *= corr; }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) p[j][e] = exp2_fast(s[j][e] - next);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) st.l[e] += p[0][e] + p[1][e];
  uint32_t vw[2 * NG];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile + 256 * NG + i * 512 + lane * 16);
    vw[4 * i] = u.x; vw[4 * i + 1] = u.y; vw[4 * i + 2] = u.z; vw[4 * i + 3] = u.w;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint32_t b0 = transpose8(pack_f16x2(p[0][0] * sv[0][g], p[0][1] * sv[0][g]));
    const uint32_t b1 = transpose8(pack_f16x2(p[1][0] * sv[1][g], p[1][1] * sv[1][g]));
    const uint32_t v0 = vw[g], v1 = vw[NG + g], w0 = v0 >> 8, w1 = v1 >> 8;
    mma_f16(st.o[g][0], v0 & 0x000f000fu, v0 & 0x00f000f0u, v1 & 0x000f000fu, v1 & 0x00f000f0u, b0, b1);
    mma_f16(st.o[g][1], w0 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x000f000fu, w1 & 0x00f000f0u, b0, b1);
    const uint32_t eight = r == g ? 0x80088008u : 0u;                                  // -8 * 2^-24 in row g
    mma_f16(st.z, eight, 0u, eight, 0u, b0, b1);
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
// than a few more tiles. Every block finds the places of its warps by a sum over the rows' lengths.
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
    rows[w] = row;
    before[w] = b * plan.units;
  }
  __syncthreads();
  return plan;
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

template <int NG> __host__ __device__ constexpr int q4_stages() { return 3; }
template <int NG> __host__ __device__ constexpr int q4_smem() { return kQ4Warps * q4_stages<NG>() * (576 + 512) * NG; }

// Each warp goes its own way through its range: a ring of shared-memory stages, each a tile and, at the start of a unit, the
// unit's query rows, filled by asynchronous copies that run ahead across units. A unit that lies within the range is finished
// from registers; parts of others go to `part` for the kernel below.
template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4Threads, NG <= 2 ? 6 : NG <= 4 ? 4 : 2) paged_decode_q4_kernel(const __grid_constant__ Q4DecodeArgs a) {
  constexpr int HD = NG * 32, TILE = 576 * NG, STAGE = TILE + 512 * NG, STAGES = q4_stages<NG>(), REC = HD + 4;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int plan_rows[kQ4Warps + 1];
  __shared__ long long plan_before[kQ4Warps + 1];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int group = a.hq / a.hkv;
  const int worker = blockIdx.x * kQ4Warps + warp;
  // rows without tokens
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (q4_len(a, row) > 0) continue;
    for (int i = threadIdx.x * 4; i < a.hq * HD; i += kQ4Threads * 4)
      q4_store4<BF16>(a.out + (size_t)row * a.out_stride + i, 0.f, 0.f, 0.f, 0.f);
  }
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
      const uint32_t into = (uint32_t)(at[i] - plan_before[warp + i]), unit = into / (uint32_t)n, off = into - unit * n;
      now.row = row;
      now.unit = unit;
      now.len = len;
      now.begin = -(int)off;
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
    const uint32_t head_bytes = a.tiles * TILE, page_bytes = a.hkv * head_bytes;
    Q4Cursor ahead = now;
    const int* page = nullptr;                   // table entry of tile `fetch`
    const uint8_t* base = nullptr;               // kv head of `ahead` in page 0, at this lane's piece
    uint32_t inside = 0;                         // byte of the tile in its page
    int fetch = 0, stage_in = 0, block = 0;
    uint32_t missing = 0;                        // stages whose page is not in the pool
    bool fresh = true;                           // tile `fetch` is the warp's first of its unit
    auto enter = [&](int t) {
      const int seq = a.seqs != nullptr ? a.seqs[ahead.row] : ahead.row;
      page = a.block_table + (size_t)seq * a.max_blocks;
      inside = 0;
      if (t > 0) {
        const int skip = t / a.tiles;
        page += skip;
        inside = (t - skip * a.tiles) * TILE;
      }
      base = a.pool + (size_t)(a.slices == 1 ? ahead.unit : ahead.unit / a.slices) * head_bytes + lane * 16;
      block = *page;
    };
    auto issue = [&]() {
      if (fetch < count) {
        const uint32_t to = to0 + stage_in * STAGE;
        if ((uint32_t)block < (uint32_t)a.num_blocks) {
          const uint8_t* from = base + ((size_t)(uint32_t)block * page_bytes + inside);
#pragma unroll
          for (int i = 0; i < TILE / 512; ++i) copy16(to + i * 512, from + i * 512);
          if (TILE % 512 != 0 && lane * 16 < TILE % 512) copy16(to + TILE / 512 * 512, from + TILE / 512 * 512);
        } else {
          missing |= 1u << stage_in;
        }
        if (fresh) {
          const int kvh = a.slices == 1 ? ahead.unit : ahead.unit / a.slices, g0 = (ahead.unit - kvh * a.slices) * 8;
          const int pieces = min(8, group - g0) * (HD / 8);
          const uint16_t* q = a.q + (size_t)ahead.row * a.q_stride + (size_t)(kvh * group + g0) * HD;
          for (int i = lane; i < pieces; i += 32) copy16(to + TILE + (i - lane) * 16, q + i * 8);
          fresh = false;
        }
        if (++fetch < count) {
          if (fetch == ahead.end) {
            ahead.next(a, plan.units);
            enter(0);
            fresh = true;
          } else {
            inside += TILE;
            if (inside == head_bytes) {
              inside = 0;
              block = *++page;
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
    };
    enter(-ahead.begin);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue();

    Q4Query<NG> f;
    Q4State<NG> st;
    int mine = 0, stage = 0;
    for (;;) {
      const int kvh = a.slices == 1 ? now.unit : now.unit / a.slices, g0 = (now.unit - kvh * a.slices) * 8;
      const int heads = min(8, group - g0), head0 = kvh * group + g0;
      st.clear();
      const int stop = min(now.end, count);
      for (bool first = true; mine < stop; ++mine, first = false) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                            // all lanes' pieces have landed; the previous stage has been read
        const uint8_t* tile = ring + stage * STAGE;
        if (first) q4_load_query<NG, BF16>(f, tile + TILE, heads, a.scale);
        issue();
        if (missing >> stage & 1) missing &= ~(1u << stage);
        else q4_tile<NG>(st, f, tile, now.len - (mine - now.begin) * kQ4Tile);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
      }
      // ---- the unit, or the warp's part of it
      const bool begins = now.begin >= 0, ends = now.end <= count;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], off);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 2 * c + e;
        const bool whole = begins && ends;
        // slot 0: the unit began before this range; slot 1: it goes on after it
        float* rec = a.part + (((size_t)worker * 2 + (begins ? 1 : 0)) * a.heads + h) * REC;
        const float by = !whole ? 16777216.f : st.l[e] == 0.f ? 0.f : 16777216.f / st.l[e];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float z = __shfl_sync(0xffffffffu, st.z[e], 4 * g + c);
          const float4 o = make_float4((st.o[g][0][e] + z) * by, fmaf(st.o[g][0][2 + e], 0.0625f, z) * by,
                                       (st.o[g][1][e] + z) * by, fmaf(st.o[g][1][2 + e], 0.0625f, z) * by);
          if (h >= heads) continue;
          if (whole) q4_store4<BF16>(a.out + (size_t)now.row * a.out_stride + (size_t)(head0 + h) * HD + 32 * g + 4 * r, o.x, o.y, o.z, o.w);
          else *reinterpret_cast<float4*>(rec + 32 * g + 4 * r) = o;
        }
        if (!whole && h < heads && r == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(st.m[e], st.l[e]);
      }
      if (begins && !ends) owner = make_int4(now.row, now.unit, (int)((start + now.end - 1) / plan.per), 0);
      if (now.end >= count) break;
      now.next(a, plan.units);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  if (lane == 0) a.owner[worker] = owner;
}
// Joins the parts of units that several warps share: slot 1 of the warp that began it, slot 0 of the others. Block x looks after
// four workers' units. SPREAD: few long units; block (x, y) does head y, its groups of HD / 4 threads take turns with the records
// and meet in shared memory. Otherwise a group of threads does all records of a unit's head by itself.
constexpr int kQ4MergeThreads = 256;

template <int NG, bool BF16, bool SPREAD>
__global__ void __launch_bounds__(kQ4MergeThreads) paged_decode_q4_merge_kernel(const __grid_constant__ Q4DecodeArgs a) {
  constexpr int HD = NG * 32, REC = HD + 4, LANES = HD / 4, SETS = kQ4MergeThreads / LANES;
  __shared__ __align__(16) float sm_o[SPREAD ? SETS : 1][HD];
  __shared__ float sm_m[SETS], sm_l[SETS];
  const int set = threadIdx.x / LANES, d = (threadIdx.x - set * LANES) * 4, group = a.hq / a.hkv;
  // every block waits, also one without work: what follows this kernel follows the attention kernel too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int4 owners[kQ4Warps];
#pragma unroll
  for (int i = 0; i < kQ4Warps; ++i) owners[i] = a.owner[blockIdx.x * kQ4Warps + i];
#pragma unroll
  for (int i = 0; i < kQ4Warps; ++i) {
    if (owners[i].x < 0) continue;
    const int row = owners[i].x, unit = owners[i].y, last = owners[i].z, worker = blockIdx.x * kQ4Warps + i;
    const int kvh = unit / a.slices, g0 = (unit - kvh * a.slices) * 8, heads = min(8, group - g0);
    const int step = SPREAD ? (int)gridDim.y : SETS;
    for (int h = SPREAD ? blockIdx.y : set < SETS ? set : heads; h < heads; h += step) {
      float top = kQ4None, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (set < SETS) {
#pragma unroll 4
        for (int w = worker + (SPREAD ? set : 0); w <= last; w += SPREAD ? SETS : 1) {
          const float* rec = a.part + (((size_t)w * 2 + (w == worker ? 1 : 0)) * a.heads + h) * REC;
          const float2 ml = *reinterpret_cast<const float2*>(rec + HD);
          const float4 o = *reinterpret_cast<const float4*>(rec + d);
          const float next = fmaxf(top, ml.x), x = exp2_fast(top - next), y = exp2_fast(ml.x - next);
          sum = sum * x + ml.y * y;
          acc.x = acc.x * x + o.x * y; acc.y = acc.y * x + o.y * y; acc.z = acc.z * x + o.z * y; acc.w = acc.w * x + o.w * y;
          top = next;
        }
      }
      if (SPREAD) {
        __syncthreads();
        if (set < SETS) {
          *reinterpret_cast<float4*>(&sm_o[set][d]) = acc;
          if (d == 0) { sm_m[set] = top; sm_l[set] = sum; }
        }
        __syncthreads();
        if (set > 0) continue;
        float all = kQ4None;
#pragma unroll
        for (int s = 0; s < SETS; ++s) all = fmaxf(all, sm_m[s]);
        sum = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          const float x = exp2_fast(sm_m[s] - all);
          const float4 v = *reinterpret_cast<const float4*>(&sm_o[s][d]);
          sum += sm_l[s] * x;
          acc.x += v.x * x; acc.y += v.y * x; acc.z += v.z * x; acc.w += v.w * x;
        }
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      q4_store4<BF16>(a.out + (size_t)row * a.out_stride + (size_t)(kvh * group + g0 + h) * HD + d, acc.x * inv, acc.y * inv,
                      acc.z * inv, acc.w * inv);
    }
  }
}

// Blocks of the attention kernel that the GPU holds at a time: the most of a call.
template <int NG, bool BF16>
static int q4_blocks() {
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  int& n = known[dev];
  if (n == 0) {
    int per_sm = 0;
    auto k = paged_decode_q4_kernel<NG, BF16>;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, q4_smem<NG>()) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, kQ4Threads, q4_smem<NG>()) != cudaSuccess || per_sm < 1)
      return -1;
    n = per_sm * num_sms();
  }
  return n;
}

template <int NG, bool BF16>
static int launch_q4_decode(const Q4DecodeArgs& a, int blocks, cudaStream_t st) {
  if (blocks > q4_blocks<NG, BF16>()) return -5;
  paged_decode_q4_kernel<NG, BF16><<<blocks, kQ4Threads, q4_smem<NG>(), st>>>(a);
  // starts while the attention kernel runs out
  const bool spread = (long long)a.rows * a.hkv * a.slices * 8 < (long long)blocks * kQ4Warps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, spread ? a.heads : 1);
  cfg.blockDim = dim3(kQ4MergeThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = spread ? cudaLaunchKernelEx(&cfg, paged_decode_q4_merge_kernel<NG, BF16, true>, a)
                               : cudaLaunchKernelEx(&cfg, paged_decode_q4_merge_kernel<NG, BF16, false>, a);
  if (e != cudaSuccess) return -(int)e;
  return check_launch("paged_decode_q4");
}

}  // namespace icb

using namespace icb;

// The most blocks of icb_paged_decode_q4 for a head size; negative: not covered.
ICB_API int icb_paged_decode_q4_blocks(int hd, int dtype) {
  const bool bf = dtype == kBF16;
  switch (hd) {
    case 64: return bf ? q4_blocks<2, true>() : q4_blocks<2, false>();
    case 128: return bf ? q4_blocks<4, true>() : q4_blocks<4, false>();
    case 192: return bf ? q4_blocks<6, true>() : q4_blocks<6, false>();
    case 256: return bf ? q4_blocks<8, true>() : q4_blocks<8, false>();
  }
  return -3;
}

// q: [rows, hq * hd] 16-bit rows of pitch q_stride (16-byte aligned); pool: num_blocks pages of [hkv][tiles] tiles; row i
// attends over the first lens[i] tokens of table row seqs[i] (null: i). out: [rows, out_stride], same type. hd 64, 128, 192
// or 256. scratch: blocks * 4 * (4 + 2 * min(8, hq / hkv) * (hd + 4)) floats, 16-byte aligned.
ICB_API int icb_paged_decode_q4(const void* q, long long q_stride, const void* pool, const int* block_table, const int* seqs,
                                const int* lens, void* out, long long out_stride, void* scratch, int rows, int hq, int hkv,
                                int hd, int tiles, int max_blocks, int table_rows, int num_blocks, int blocks, float scale,
                                int dtype, void* stream) {
  if (rows <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || tiles < 1 || blocks < 1 || q_stride % 8) return -2;
  const int slices = (hq / hkv + 7) / 8;
  // offsets within a page and within a row's units are 32-bit
  if ((long long)hkv * tiles * 18 * hd > 0x7fffffffLL || (long long)max_blocks * tiles * hkv * slices > 0x7fffffffLL ||
      (long long)max_blocks * tiles > 0x7ffffffLL)
    return -2;
  Q4DecodeArgs a{reinterpret_cast<const uint16_t*>(q), q_stride, reinterpret_cast<const uint8_t*>(pool), block_table, seqs,
                 lens, reinterpret_cast<uint16_t*>(out), out_stride, reinterpret_cast<int4*>(scratch),
                 reinterpret_cast<float*>(scratch) + (size_t)blocks * kQ4Warps * 4, rows, hq, hkv, slices,
                 hq / hkv < 8 ? hq / hkv : 8, tiles, max_blocks, table_rows, num_blocks, scale * kLog2e};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == kBF16;
  if (!bf && dtype != kF16) return -4;
  switch (hd) {
    case 64: return bf ? launch_q4_decode<2, true>(a, blocks, st) : launch_q4_decode<2, false>(a, blocks, st);
    case 128: return bf ? launch_q4_decode<4, true>(a, blocks, st) : launch_q4_decode<4, false>(a, blocks, st);
    case 192: return bf ? launch_q4_decode<6, true>(a, blocks, st) : launch_q4_decode<6, false>(a, blocks, st);
    case 256: return bf ? launch_q4_decode<8, true>(a, blocks, st) : launch_q4_decode<8, false>(a, blocks, st);
  }
  return -3;
}
