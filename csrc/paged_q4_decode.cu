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
//     side a matrix instruction with a constant operand sums -8 p_t sv_tg from the same rounded products.
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
constexpr int kQ4MinTiles = kQ4Warps;           // a worker has at least a tile for each warp
constexpr float kQ4Top = 12.f;                  // log2 of the largest fp16 probability times scale right after a new maximum
constexpr float kQ4Slack = 3.f;                 // and how far it may grow before the maximum is taken again: 2^15 fits fp16
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
  float* part;                  // [workers][2][8] records of HD + 4 floats: outputs, maximum, sum
  int rows, hq, hkv, slices, tiles, max_blocks, table_rows, num_blocks, workers;
  uint32_t tiles_inverse;       // ceil(2^32 / tiles)
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
__device__ __forceinline__ void copy16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
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
  float z[NG][4];               // -8 * sum of the rounded p * value scale, in the units of o
  float m[2], l[2];             // what is subtracted for heads 2c, 2c + 1 (equal in all lanes r), this lane's sum of p
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[g][0][i] = o[g][1][i] = z[g][i] = 0.f;
    }
    m[0] = m[1] = -INFINITY;
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
  {
    uint32_t kw[2 * NG];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint4 u = *reinterpret_cast<const uint4*>(tile + p * 512 + lane * 16);
      kw[4 * p] = u.x; kw[4 * p + 1] = u.y; kw[4 * p + 2] = u.z; kw[4 * p + 3] = u.w;
    }
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
  }
  if (live < kQ4Tile) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = NG / 2; g < NG; ++g) sc[j][g] = r + 8 * j < live ? sc[j][g] : 0u;
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
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j][e] *= f.factor[e];
  }
  if (live < kQ4Tile) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (r + 8 * j >= live) s[j][0] = s[j][1] = -INFINITY;
  }
  const float top0 = fmaxf(s[0][0] + reach[0], s[1][0] + reach[1]), top1 = fmaxf(s[0][1] + reach[0], s[1][1] + reach[1]);
  // m is kQ4Top below the maximum at which it was taken
  if (__any_sync(0xffffffffu, top0 > st.m[0] + (kQ4Top + kQ4Slack) || top1 > st.m[1] + (kQ4Top + kQ4Slack))) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = e ? top1 : top0;
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float next = fmaxf(st.m[e], top - kQ4Top);
      const float corr = st.m[e] == -INFINITY ? 0.f : exp2_fast(st.m[e] - next);
      st.m[e] = next;
      st.l[e] *= corr;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        st.z[g][e] *= corr;
        st.z[g][2 + e] *= corr;
#pragma unroll
        for (int t = 0; t < 2; ++t) { st.o[g][t][e] *= corr; st.o[g][t][2 + e] *= corr; }
      }
    }
  }
  float p[2][2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float base = st.m[e] == -INFINITY ? 0.f : st.m[e];
#pragma unroll
    for (int j = 0; j < 2; ++j) p[j][e] = exp2_fast(s[j][e] - base);
    st.l[e] += p[0][e] + p[1][e];
  }
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
    mma_f16(st.z[g], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0, b1);      // -8 and -8 * 16, times 2^-24
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
// units in one line that is cut into `active` equal ranges. Every block finds its place by a sum over the rows' lengths.
struct Q4Plan {
  long long total;              // tiles of the call
  int active;                   // workers with a range
  int units;                    // units of a row
  int row;                      // row that holds tile `at`, and the tiles before that row
  long long before;
  __device__ __forceinline__ long long start(int worker) const { return total * worker / active; }
};

// `at` is the worker whose first tile is looked for. All threads of the block take part; shared: 2 * kQ4Warps + 4 words of 8.
__device__ __forceinline__ Q4Plan q4_plan(const Q4DecodeArgs& a, int worker, long long* shared) {
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
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  long long before = sum - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kQ4Warps; ++w) {
    if (w < warp) before += shared[w];
    all += shared[w];
  }
  Q4Plan plan;
  plan.units = a.hkv * a.slices;
  plan.total = all * plan.units;
  plan.active = (int)min((long long)a.workers, max(1LL, plan.total / kQ4MinTiles));
  plan.row = 0;
  plan.before = 0;
  if (worker < plan.active && plan.total > 0) {
    const long long at = plan.start(worker);
    if (at >= before * plan.units && at < (before + mine) * plan.units) {
      int row = first;
      for (; row < last; ++row) {
        const int n = q4_count(q4_len(a, row));
        if (at < (before + n) * plan.units) break;
        before += n;
      }
      shared[kQ4Warps] = row;
      shared[kQ4Warps + 1] = before * plan.units;
    }
    __syncthreads();
    plan.row = (int)shared[kQ4Warps];
    plan.before = shared[kQ4Warps + 1];
  }
  return plan;
}

// A place in the line of tiles, relative to the worker's first.
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

template <int NG> __host__ __device__ constexpr int q4_stages() { return NG <= 4 ? 4 : 3; }
template <int NG> __host__ __device__ constexpr int q4_smem() {
  return kQ4Warps * q4_stages<NG>() * 576 * NG + (kQ4Warps * 8 * (NG * 32 + 4) + kQ4Warps * 16) * 4;
}

template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4Threads, NG <= 2 ? 6 : NG <= 4 ? 4 : 2) paged_decode_q4_kernel(const __grid_constant__ Q4DecodeArgs a) {
  constexpr int HD = NG * 32, TILE = 576 * NG, STAGES = q4_stages<NG>(), REC = HD + 4;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ long long plan_words[kQ4Warps + 2];
  float* sm_o = reinterpret_cast<float*>(smem + kQ4Warps * STAGES * TILE);          // [warp][8][HD + 4]
  float* sm_m = sm_o + kQ4Warps * 8 * REC;                                          // [warp][8]
  float* sm_l = sm_m + kQ4Warps * 8;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int group = a.hq / a.hkv;
  // rows without tokens
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (q4_len(a, row) > 0) continue;
    for (int i = threadIdx.x * 4; i < a.hq * HD; i += kQ4Threads * 4)
      q4_store4<BF16>(a.out + (size_t)row * a.out_stride + i, 0.f, 0.f, 0.f, 0.f);
  }
  const Q4Plan plan = q4_plan(a, blockIdx.x, plan_words);
  if (plan.total == 0 || (int)blockIdx.x >= plan.active) return;
  const long long lo = plan.start(blockIdx.x);
  const int count = (int)(plan.start(blockIdx.x + 1) - lo);
  Q4Cursor now;
  now.row = plan.row;
  now.len = q4_len(a, now.row);
  {
    const int n = q4_count(now.len);
    const long long into = lo - plan.before;
    now.unit = (int)(into / n);
    now.begin = -(int)(into - (long long)now.unit * n);
    now.end = now.begin + n;
  }
  // ---- copies: each warp takes every fourth tile of the range and keeps STAGES - 1 of them on the way
  uint8_t* ring = smem + warp * STAGES * TILE;
  Q4Cursor ahead = now;
  int fetch = warp, stage_in = 0;
  uint32_t missing = 0;                          // stages whose page is not in the pool
  int block = -1, inside = 0;
  auto locate = [&]() {                          // page of tile `fetch`
    while (fetch >= ahead.end && fetch < count) ahead.next(a, plan.units);
    if (fetch < count) {
      const int t = fetch - ahead.begin;
      const int page = a.tiles == 1 ? t : (int)__umulhi((uint32_t)t, a.tiles_inverse);
      inside = t - page * a.tiles;
      const int seq = a.seqs != nullptr ? a.seqs[ahead.row] : ahead.row;
      block = a.block_table[(size_t)seq * a.max_blocks + page];
    }
  };
  auto issue = [&]() {
    if (fetch < count) {
      const bool ok = block >= 0 && block < a.num_blocks;
      missing = ok ? missing & ~(1u << stage_in) : missing | (1u << stage_in);
      if (ok) {
        const int kvh = a.slices == 1 ? ahead.unit : ahead.unit / a.slices;
        const uint8_t* from = a.pool + (((size_t)block * a.hkv + kvh) * a.tiles + inside) * TILE + lane * 16;
        uint8_t* to = ring + stage_in * TILE + lane * 16;
#pragma unroll
        for (int i = 0; i < TILE / 512; ++i) copy16(to + i * 512, from + i * 512);
        if (TILE % 512 != 0 && lane * 16 < TILE % 512) copy16(to + TILE / 512 * 512, from + TILE / 512 * 512);
      }
      fetch += kQ4Warps;
      locate();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
  };
  locate();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue();

  Q4Query<NG> f;
  Q4State<NG> st;
  int mine = warp, stage = 0;
  for (;;) {
    const int kvh = now.unit / a.slices, g0 = (now.unit - kvh * a.slices) * 8;
    const int heads = min(8, group - g0), head0 = kvh * group + g0;
    q4_load_query<NG, BF16>(f, a.q + (size_t)now.row * a.q_stride + (size_t)head0 * HD, heads, a.scale);
    st.clear();
    const int stop = min(now.end, count);
    for (; mine < stop; mine += kQ4Warps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();                              // all lanes' pieces have landed; the previous stage has been read
      const bool gone = missing >> stage & 1;
      issue();
      if (!gone) q4_tile<NG>(st, f, ring + stage * TILE, now.len - (mine - now.begin) * kQ4Tile);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    // ---- the warps meet: factors and sums first
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], off);
      if (st.l[e] != st.l[e] && st.m[e] == -INFINITY) st.m[e] = 0.f;         // NaN scores only: not to be taken for no tokens
    }
    __syncthreads();                             // the previous unit's records have been read
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (r == 0) { sm_m[warp * 8 + 2 * c + e] = st.m[e]; sm_l[warp * 8 + 2 * c + e] = st.l[e]; }
#pragma unroll
      for (int g = 0; g < NG; ++g)
        *reinterpret_cast<float4*>(sm_o + (warp * 8 + 2 * c + e) * REC + 32 * g + 4 * r) =
            make_float4((st.o[g][0][e] + st.z[g][e]) * 16777216.f, (st.o[g][0][2 + e] + st.z[g][2 + e]) * 1048576.f,
                        (st.o[g][1][e] + st.z[g][e]) * 16777216.f, (st.o[g][1][2 + e] + st.z[g][2 + e]) * 1048576.f);
    }
    __syncthreads();
    const bool whole = now.begin >= 0 && now.end <= count;
    for (int i = threadIdx.x; i < heads * (HD / 4); i += kQ4Threads) {
      const int h = i / (HD / 4), d = (i - h * (HD / 4)) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kQ4Warps; ++w) top = fmaxf(top, sm_m[w * 8 + h]);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kQ4Warps; ++w) {
        const float m = sm_m[w * 8 + h];
        if (m == -INFINITY) continue;
        const float x = exp2_fast(m - top);
        const float4 o = *reinterpret_cast<const float4*>(sm_o + (w * 8 + h) * REC + d);
        sum += sm_l[w * 8 + h] * x;
        acc.x += o.x * x; acc.y += o.y * x; acc.z += o.z * x; acc.w += o.w * x;
      }
      if (whole) {
        const float inv = top == -INFINITY ? 0.f : 1.f / sum;
        q4_store4<BF16>(a.out + (size_t)now.row * a.out_stride + (size_t)(head0 + h) * HD + d, acc.x * inv, acc.y * inv,
                        acc.z * inv, acc.w * inv);
      } else {
        // slot 0: the unit began before this range; slot 1: it goes on after it
        float* rec = a.part + (((size_t)blockIdx.x * 2 + (now.begin < 0 ? 0 : 1)) * 8 + h) * REC;
        *reinterpret_cast<float4*>(rec + d) = acc;
        if (d == 0) { rec[HD] = top; rec[HD + 1] = sum; }
      }
    }
    if (now.end >= count) break;
    now.next(a, plan.units);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Units that several workers share. Grid (worker, head of the slice): block (w, h) joins the unit in whose inside worker w
// starts, if no earlier worker starts inside it too. Records: slot 1 of the worker that began it, slot 0 of the others.
template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4Threads) paged_decode_q4_merge_kernel(const __grid_constant__ Q4DecodeArgs a) {
  constexpr int HD = NG * 32, REC = HD + 4, LANES = HD / 4, SETS = kQ4Threads / LANES;
  __shared__ long long plan_words[kQ4Warps + 2];
  __shared__ __align__(16) float sm_o[SETS][HD];
  __shared__ float sm_m[SETS], sm_l[SETS];
  const int worker = blockIdx.x + 1, h = blockIdx.y;
  const Q4Plan plan = q4_plan(a, worker, plan_words);
  // every block waits, also one without work: what follows this kernel follows the attention kernel too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (plan.total == 0 || worker >= plan.active) return;
  const int n = q4_count(q4_len(a, plan.row));
  const long long at = plan.start(worker), into = at - plan.before;
  const int unit = (int)(into / n);
  const long long begin = plan.before + (long long)unit * n, end = begin + n;
  if (begin == at || plan.start(worker - 1) > begin) return;
  const int kvh = unit / a.slices, g0 = (unit - kvh * a.slices) * 8, group = a.hq / a.hkv;
  if (h >= min(8, group - g0)) return;
  // sets of HD / 4 threads take every SETS-th record
  const int set = threadIdx.x / LANES, d = (threadIdx.x - set * LANES) * 4;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (set < SETS) {
    for (int w = worker - 1 + set; w < plan.active && plan.start(w) < end; w += SETS) {
      const float* rec = a.part + (((size_t)w * 2 + (w < worker ? 1 : 0)) * 8 + h) * REC;
      const float m = rec[HD], l = rec[HD + 1];
      const float4 o = *reinterpret_cast<const float4*>(rec + d);
      if (m == -INFINITY) continue;
      const float next = fmaxf(top, m), x = top == -INFINITY ? 0.f : exp2_fast(top - next), y = exp2_fast(m - next);
      sum = sum * x + l * y;
      acc.x = acc.x * x + o.x * y; acc.y = acc.y * x + o.y * y; acc.z = acc.z * x + o.z * y; acc.w = acc.w * x + o.w * y;
      top = next;
    }
    *reinterpret_cast<float4*>(&sm_o[set][d]) = acc;
    if (d == 0) { sm_m[set] = top; sm_l[set] = sum; }
  }
  __syncthreads();
  for (int e = threadIdx.x * 4; e < HD; e += kQ4Threads * 4) {
    float all = -INFINITY, total = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < SETS; ++s) all = fmaxf(all, sm_m[s]);
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      if (sm_m[s] == -INFINITY) continue;
      const float x = exp2_fast(sm_m[s] - all);
      const float4 v = *reinterpret_cast<const float4*>(&sm_o[s][e]);
      total += sm_l[s] * x;
      o.x += v.x * x; o.y += v.y * x; o.z += v.z * x; o.w += v.w * x;
    }
    const float inv = all == -INFINITY ? 0.f : 1.f / total;
    q4_store4<BF16>(a.out + (size_t)plan.row * a.out_stride + (size_t)(kvh * group + g0 + h) * HD + e, o.x * inv, o.y * inv,
                    o.z * inv, o.w * inv);
  }
}

// Blocks of the attention kernel that the GPU holds at a time: the most workers of a call.
template <int NG, bool BF16>
static int q4_workers() {
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
static int launch_q4_decode(Q4DecodeArgs& a, int workers, cudaStream_t st) {
  const int most = q4_workers<NG, BF16>();
  if (most < 1) return -5;
  a.workers = min(workers, most);
  paged_decode_q4_kernel<NG, BF16><<<a.workers, kQ4Threads, q4_smem<NG>(), st>>>(a);
  if (a.workers > 1) {
    // starts while the attention kernel runs, finds its units, waits for the records
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.workers - 1, min(8, a.hq / a.hkv));
    cfg.blockDim = dim3(kQ4Threads);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_q4_merge_kernel<NG, BF16>, (const Q4DecodeArgs)a);
    if (e != cudaSuccess) return -(int)e;
  }
  return check_launch("paged_decode_q4");
}

}  // namespace icb

using namespace icb;

// The most workers of icb_paged_decode_q4 for a head size; negative: not covered.
ICB_API int icb_paged_decode_q4_workers(int hd, int dtype) {
  const bool bf = dtype == kBF16;
  switch (hd) {
    case 64: return bf ? q4_workers<2, true>() : q4_workers<2, false>();
    case 128: return bf ? q4_workers<4, true>() : q4_workers<4, false>();
    case 192: return bf ? q4_workers<6, true>() : q4_workers<6, false>();
    case 256: return bf ? q4_workers<8, true>() : q4_workers<8, false>();
  }
  return -3;
}

// q: [rows, hq * hd] 16-bit rows of pitch q_stride (16-byte aligned); pool: num_blocks pages of [hkv][tiles] tiles; row i
// attends over the first lens[i] tokens of table row seqs[i] (null: i). out: [rows, out_stride], same type. hd 64, 128, 192
// or 256. scratch: workers * 16 * (hd + 4) floats.
ICB_API int icb_paged_decode_q4(const void* q, long long q_stride, const void* pool, const int* block_table, const int* seqs,
                                const int* lens, void* out, long long out_stride, void* scratch, int rows, int hq, int hkv,
                                int hd, int tiles, int max_blocks, int table_rows, int num_blocks, int workers, float scale,
                                int dtype, void* stream) {
  if (rows <= 0) return 0;
  if (hkv < 1 || hq < 1 || hq % hkv || tiles < 1 || workers < 1 || q_stride % 8 || (long long)max_blocks * tiles > (1LL << 26)) return -2;
  Q4DecodeArgs a{reinterpret_cast<const uint16_t*>(q), q_stride, reinterpret_cast<const uint8_t*>(pool), block_table, seqs,
                 lens, reinterpret_cast<uint16_t*>(out), out_stride, reinterpret_cast<float*>(scratch), rows, hq, hkv,
                 (hq / hkv + 7) / 8, tiles, max_blocks, table_rows, num_blocks, workers,
                 (uint32_t)(((1ULL << 32) + tiles - 1) / tiles), scale * kLog2e};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == kBF16;
  if (!bf && dtype != kF16) return -4;
  switch (hd) {
    case 64: return bf ? launch_q4_decode<2, true>(a, workers, st) : launch_q4_decode<2, false>(a, workers, st);
    case 128: return bf ? launch_q4_decode<4, true>(a, workers, st) : launch_q4_decode<4, false>(a, workers, st);
    case 192: return bf ? launch_q4_decode<6, true>(a, workers, st) : launch_q4_decode<6, false>(a, workers, st);
    case 256: return bf ? launch_q4_decode<8, true>(a, workers, st) : launch_q4_decode<8, false>(a, workers, st);
  }
  return -3;
}
