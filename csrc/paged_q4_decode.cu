// Attention of single query rows over the 4-bit paged cache (format: q4.cuh) on sm_100a.
//
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q . k_t),  k_td = sk_tg (n_td - 8),  v_td = sv_tg (m_td - 8)
//
// Up to eight query heads of a kv head's group are the N dimension of mma.sync.m16n8k16 (fp16, fp32 sums), 16 tokens the M
// dimension of K Q^T and 16 elements that of V^T P^T: every row of the matrix instructions is used.
//   * A code needs no conversion: four bits at the bottom of an fp16 are the number n 2^-24, exact in the matrix
//     instruction, so a word & 0x000f000f is two operands, & 0x00f000f0 two more that are 16 n 2^-24. The factor 16 is taken
//     out of the query elements beforehand and out of the output rows at the end; shifted by 8 the word gives the other four.
//   * The -8 enters through the first addend: q . (n - 8) = q . n - 8 sum q per group, a constant of the query. On the value
//     side -8 sum_t p_t sv_tg is added once at the end.
//   * The scale of a group multiplies a finished dot product (keys) or the probability before it is rounded to fp16 (values).
//   * Queries are scaled per head by a power of two to [2^14, 2^15) so that bf16 fits fp16: an element loses bits only below
//     2^-24 of the head's largest.
//   * p_t sv_tg is rounded to fp16 too. Its range is held by the maximum that the softmax subtracts: it runs over
//     log2 p_t + log2 max_g |sv_tg| instead of log2 p_t, so that the largest product is 2^14, whatever the values' magnitude.
//     Relative error 2^-11 down to 2^-28 of the largest contribution; sums, maxima and p itself stay in fp32.
// Tokens outside the sequence get probability and value scale zero by selection, so nothing stale in a page (NaN scales
// included) reaches a result. A page number outside the pool counts as a page outside the sequence.
#include "host_common.h"
#include "ptx.cuh"
#include "q4.cuh"

namespace icb {

constexpr int kQ4Warps = 4;
constexpr float kQ4Top = 14.f;                  // log2 of the largest fp16 probability times scale
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
  float* part;                  // [rows * hq, nsplit] records of HD + 2 floats when nsplit > 1
  int hq, hkv, tiles, max_blocks, table_rows, num_blocks, nsplit;
  float scale;                  // score factor times log2(e)
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ void q4_store(const Q4DecodeArgs& a, int row, int head, int hd, int d, float val) {
  const size_t at = (size_t)row * a.out_stride + (size_t)head * hd + d;
  if (BF16) reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16(val);
  else reinterpret_cast<__half*>(a.out)[at] = __float2half(val);
}

// The query operand of up to eight heads, resident in registers.
template <int NG>
struct Q4Query {
  uint32_t b[NG][4];            // B fragments of the two matrix instructions of a group
  float start[NG][2];           // -8 * sum of the group's query elements (in units of 2^-24), heads 2c and 2c + 1
  float factor[2];              // from the sums to the base-2 score
};

template <int NG, bool BF16>
__device__ __forceinline__ void q4_load_query(Q4Query<NG>& f, const uint16_t* q, int heads, float scale) {
  constexpr int HD = NG * 32;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  float x[NG][8];
  float top = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (r < heads) u = *reinterpret_cast<const uint4*>(q + r * HD + g * 32 + c * 8);
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
    f.start[g][0] = __shfl_sync(0xffffffffu, sum, 8 * c);                    // head 2c: lanes 4 (2c) ..
    f.start[g][1] = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
  }
  f.factor[0] = __shfl_sync(0xffffffffu, back, 8 * c);
  f.factor[1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
}

// Running state of a warp: this lane's part of eight heads.
template <int NG>
struct Q4State {
  float o[NG][2][4];            // V^T P^T: elements 32 g + 4 r + 2 m + (reg >> 1), heads 2c + (reg & 1); odd elements times 16
  float vs[NG][2];              // sum of p * value scale over this lane's tokens
  float m[2], l[2];             // maximum of the heads 2c, 2c + 1 (equal in all lanes r), this lane's sum of p
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        o[g][t][0] = o[g][t][1] = o[g][t][2] = o[g][t][3] = 0.f;
        vs[g][t] = 0.f;
      }
    }
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
};

// One tile of 16 tokens; `live` of them belong to the sequence (16 or more: all).
template <int NG>
__device__ __forceinline__ void q4_tile(Q4State<NG>& st, const Q4Query<NG>& f, const uint8_t* tile, int live) {
  constexpr int NP = NG / 2;                     // 16-byte pieces per lane of the keys, and of the values
  const int lane = threadIdx.x & 31, r = lane >> 2;
  uint32_t kw[2 * NG], vw[2 * NG];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile + p * 512 + lane * 16);
    kw[4 * p] = u.x; kw[4 * p + 1] = u.y; kw[4 * p + 2] = u.z; kw[4 * p + 3] = u.w;
  }
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile + 256 * NG + p * 512 + lane * 16);
    vw[4 * p] = u.x; vw[4 * p + 1] = u.y; vw[4 * p + 2] = u.z; vw[4 * p + 3] = u.w;
  }
  // scales of tokens r and r + 8: NG fp16 of the keys, NG of the values
  uint32_t sc[2][NG];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint8_t* at = tile + 512 * NG + (r + 8 * j) * 4 * NG;
    if (NG == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(at);
      sc[j][0] = u.x; sc[j][1] = u.y;
    } else if (NG % 4 == 0) {
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
  const bool seen[2] = {r < live, r + 8 < live};
  if (live < kQ4Tile) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = NG / 2; g < NG; ++g) sc[j][g] = seen[j] ? sc[j][g] : 0u;
  }
  // ---- scores of tokens r, r + 8 and heads 2c, 2c + 1: s[j][e]
  float s[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float d[4] = {f.start[g][0], f.start[g][1], f.start[g][0], f.start[g][1]};
    const uint32_t a = kw[g], b = kw[NG + g];
    mma_f16(d, a & 0x000f000fu, b & 0x000f000fu, a & 0x00f000f0u, b & 0x00f000f0u, f.b[g][0], f.b[g][1]);
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
  // ---- value scales in fp32, their largest magnitude per token
  float sv[2][NG], reach[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float top = 5.9604645e-8f;                   // 2^-24: a token whose values are all zero still counts in the sum
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&sc[j][(NG + g) >> 1]));
      sv[j][g] = (g & 1) ? two.y : two.x;
      top = fmaxf(top, fabsf(sv[j][g]));
    }
    reach[j] = log2_fast(top);
  }
  float p[2][2], corr[2];
  bool moved = false;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[j][e] = live < kQ4Tile && !seen[j] ? -INFINITY : s[j][e] * f.factor[e];
      top = fmaxf(top, s[j][e] + reach[j]);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float next = fmaxf(st.m[e], top);
    moved |= next != st.m[e];
    corr[e] = st.m[e] == -INFINITY ? 0.f : exp2_fast(st.m[e] - next);
    st.m[e] = next;
    const float base = next == -INFINITY ? 0.f : next - kQ4Top;
#pragma unroll
    for (int j = 0; j < 2; ++j) p[j][e] = exp2_fast(s[j][e] - base);          // 2^14 times the probability over its reach
  }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      st.l[e] *= corr[e];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        st.vs[g][e] *= corr[e];
#pragma unroll
        for (int t = 0; t < 2; ++t) { st.o[g][t][e] *= corr[e]; st.o[g][t][2 + e] *= corr[e]; }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) st.l[e] += p[0][e] + p[1][e];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    uint32_t b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float x0 = p[j][0] * sv[j][g], x1 = p[j][1] * sv[j][g];
      st.vs[g][0] += x0;
      st.vs[g][1] += x1;
      b[j] = transpose8(pack_f16x2(x0, x1));
    }
    const uint32_t v0 = vw[g], v1 = vw[NG + g], w0 = v0 >> 8, w1 = v1 >> 8;
    mma_f16(st.o[g][0], v0 & 0x000f000fu, v0 & 0x00f000f0u, v1 & 0x000f000fu, v1 & 0x00f000f0u, b[0], b[1]);
    mma_f16(st.o[g][1], w0 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x000f000fu, w1 & 0x00f000f0u, b[0], b[1]);
  }
}

// Finished values of the warp's heads: sums of p over all lanes, outputs with the -8 and the factors taken out (still to be
// divided by the sum of p).
template <int NG>
__device__ __forceinline__ void q4_finish(Q4State<NG>& st) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], off);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) st.vs[g][e] += __shfl_xor_sync(0xffffffffu, st.vs[g][e], off);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        st.o[g][t][e] = st.o[g][t][e] * 16777216.f - 8.f * st.vs[g][e];
        st.o[g][t][2 + e] = st.o[g][t][2 + e] * (16777216.f / 16.f) - 8.f * st.vs[g][e];
      }
    }
  }
}

// Grid (row, slice of at most eight heads of a kv head, split): a split owns a contiguous range of tiles, its warps take
// turns. Partial records [HD outputs, max, sum] of (row, head, split) meet in paged_decode_q4_merge_kernel.
template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4Warps * 32) paged_decode_q4_kernel(const Q4DecodeArgs a) {
  constexpr int HD = NG * 32;
  const int row = blockIdx.x, split = blockIdx.z;
  const int group = a.hq / a.hkv, slices = (group + 7) / 8;
  const int kvh = blockIdx.y / slices, g0 = (blockIdx.y - kvh * slices) * 8;
  const int heads = min(8, group - g0), head0 = kvh * group + g0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int seq = a.seqs != nullptr ? a.seqs[row] : row;
  int ctx = min(a.lens[row], a.max_blocks * a.tiles * kQ4Tile);
  if (seq < 0 || seq >= a.table_rows) ctx = 0;
  const int* pages = a.block_table + (size_t)seq * a.max_blocks;
  const int total = (max(ctx, 0) + kQ4Tile - 1) / kQ4Tile;
  const int each = (total + a.nsplit - 1) / a.nsplit;
  const int begin = split * each, end = min(total, begin + each);
  Q4Query<NG> f;
  q4_load_query<NG, BF16>(f, a.q + (size_t)row * a.q_stride + (size_t)head0 * HD, heads, a.scale);
  Q4State<NG> st;
  st.clear();
  for (int t = begin + warp; t < end; t += kQ4Warps) {
    const int page = t / a.tiles;
    const int blk = pages[page];
    if (blk < 0 || blk >= a.num_blocks) continue;
    const uint8_t* tile = a.pool + (((size_t)blk * a.hkv + kvh) * a.tiles + (t - page * a.tiles)) * q4_tile_bytes(HD);
    q4_tile<NG>(st, f, tile, ctx - t * kQ4Tile);
  }
  q4_finish(st);
  __shared__ float sm_m[kQ4Warps][8], sm_l[kQ4Warps][8];
  __shared__ float sm_o[kQ4Warps][8][HD + 4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (r == 0) { sm_m[warp][2 * c + e] = st.m[e]; sm_l[warp][2 * c + e] = st.l[e]; }
#pragma unroll
    for (int g = 0; g < NG; ++g)
      *reinterpret_cast<float4*>(&sm_o[warp][2 * c + e][32 * g + 4 * r]) =
          make_float4(st.o[g][0][e], st.o[g][0][2 + e], st.o[g][1][e], st.o[g][1][2 + e]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * HD; i += blockDim.x) {
    const int h = i / HD, d = i - h * HD;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kQ4Warps; ++w) mm = fmaxf(mm, sm_m[w][h]);
    float ll = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kQ4Warps; ++w) {
      if (sm_m[w][h] == -INFINITY) continue;
      const float x = exp2_fast(sm_m[w][h] - mm);
      ll += sm_l[w][h] * x;
      acc += sm_o[w][h][d] * x;
    }
    if (a.nsplit == 1) {
      q4_store<BF16>(a, row, head0 + h, HD, d, mm == -INFINITY ? 0.f : acc / ll);
    } else {
      float* rec = a.part + (((size_t)row * a.hq + head0 + h) * a.nsplit + split) * (HD + 2);
      rec[d] = acc;
      if (d == 0) { rec[HD] = mm; rec[HD + 1] = ll; }
    }
  }
}

template <int NG, bool BF16>
__global__ void paged_decode_q4_merge_kernel(const Q4DecodeArgs a) {
  constexpr int HD = NG * 32;
  const int row = blockIdx.x / a.hq, head = blockIdx.x - row * a.hq, d = threadIdx.x;
  const float* rec = a.part + (size_t)blockIdx.x * a.nsplit * (HD + 2);
  float mm = -INFINITY;
  for (int s = 0; s < a.nsplit; ++s) mm = fmaxf(mm, rec[s * (HD + 2) + HD]);
  float ll = 0.f, acc = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float ms = rec[s * (HD + 2) + HD];
    if (ms == -INFINITY) continue;
    const float x = exp2_fast(ms - mm);
    ll += rec[s * (HD + 2) + HD + 1] * x;
    acc += rec[s * (HD + 2) + d] * x;
  }
  q4_store<BF16>(a, row, head, HD, d, mm == -INFINITY ? 0.f : acc / ll);
}

template <int NG, bool BF16>
static int launch_q4_decode(const Q4DecodeArgs& a, int rows, cudaStream_t st) {
  const int slices = (a.hq / a.hkv + 7) / 8;
  paged_decode_q4_kernel<NG, BF16><<<dim3(rows, a.hkv * slices, a.nsplit), kQ4Warps * 32, 0, st>>>(a);
  if (a.nsplit > 1) paged_decode_q4_merge_kernel<NG, BF16><<<rows * a.hq, NG * 32, 0, st>>>(a);
  return check_launch("paged_decode_q4");
}

}  // namespace icb

using namespace icb;

// q: [rows, hq * hd] 16-bit rows of pitch q_stride (16-byte aligned); pool: num_blocks pages of [hkv][tiles] tiles; row i
// attends over the first lens[i] tokens of table row seqs[i] (null: i). out: [rows, out_stride], same type. hd 64, 128, 192
// or 256. scratch: rows * hq * nsplit * (hd + 2) floats when nsplit > 1.
ICB_API int icb_paged_decode_q4(const void* q, long long q_stride, const void* pool, const int* block_table, const int* seqs,
                                const int* lens, void* out, long long out_stride, void* scratch, int rows, int hq, int hkv,
                                int hd, int tiles, int max_blocks, int table_rows, int num_blocks, int nsplit, float scale,
                                int dtype, void* stream) {
  if (rows <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || tiles < 1 || nsplit < 1 || q_stride % 8 || hkv * ((hq / hkv + 7) / 8) > 65535) return -2;
  Q4DecodeArgs a{reinterpret_cast<const uint16_t*>(q), q_stride, reinterpret_cast<const uint8_t*>(pool), block_table, seqs,
                 lens, reinterpret_cast<uint16_t*>(out), out_stride, reinterpret_cast<float*>(scratch), hq, hkv, tiles,
                 max_blocks, table_rows, num_blocks, nsplit, scale * kLog2e};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == kBF16;
  if (!bf && dtype != kF16) return -4;
  switch (hd) {
    case 64: return bf ? launch_q4_decode<2, true>(a, rows, st) : launch_q4_decode<2, false>(a, rows, st);
    case 128: return bf ? launch_q4_decode<4, true>(a, rows, st) : launch_q4_decode<4, false>(a, rows, st);
    case 192: return bf ? launch_q4_decode<6, true>(a, rows, st) : launch_q4_decode<6, false>(a, rows, st);
    case 256: return bf ? launch_q4_decode<8, true>(a, rows, st) : launch_q4_decode<8, false>(a, rows, st);
  }
  return -3;
}
