// Rows of the 4-bit paged key / value cache (format: q4.cuh): quantise and write, read back.
//
// Quantisation of a group of 32 elements: scale = m / -8 rounded to fp16, m the element of largest magnitude (the largest
// if the smallest is as far from zero), so that m itself is code 0 and the other end of the range reaches code 15;
// n = clamp(round(x / scale), -8, 7) + 8, ties to even.
//
// Rounding without a division: x and scale have at most 11 significant bits, so x / scale is either a tie k + 1/2 or differs
// from one by at least 2^-15 of its value, 2^-16 or more. y = x * (1 / scale) with the correctly rounded reciprocal is off by
// at most 2^-21 (|y| <= 8), and fma(x, 1 / scale, 48) rounds it to a multiple of 2^-18: ties come out as ties, everything else
// stays on its side of them. Adding 1.5 * 2^23 - 40 then rounds to an integer, ties to even, whose low bits are the code.
//
// Both directions are bound by memory. Two forms each: one thread per 8 elements of a row, for few rows; and one warp per tile
// of 16 rows and head in the order of the tile's lanes, so that all 18 hd bytes of the tile leave or arrive in 512-byte pieces
// (a row by itself touches all of a tile's value sectors, two bytes in each). Rows that do not fill a tile go one by one.
#include "host_common.h"
#include "ptx.cuh"
#include "q4.cuh"

namespace icb {

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <bool BF16>
__device__ __forceinline__ void widen8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = BF16 ? unpack_bf16x2(w[i]) : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Scale of a group from its extremes; a NaN among the elements makes it NaN.
__device__ __forceinline__ __half q4_scale(float most, float least) {
  float s = (most >= -least ? most : least) * -0.125f;
  if (s > 65504.f) s = 65504.f;
  if (s < -65504.f) s = -65504.f;
  const __half h = __float2half_rn(s);
  return __half2float(h) == 0.f ? __ushort_as_half(0) : h;    // no negative zero
}

struct Q4Scale {
  __half half;
  float inv;
  bool plain;                   // the largest element is -8 scales exactly: no code can be below 0
};
__device__ __forceinline__ Q4Scale q4_group(float most, float least) {
  Q4Scale s;
  s.half = q4_scale(most, least);
  const float scale = __half2float(s.half), m = most >= -least ? most : least;
  s.inv = scale != 0.f ? __frcp_rn(scale) : 0.f;
  s.plain = scale * -8.f == m;
  return s;
}

// N codes (at most 8) of a group, lowest nibble first.
template <int N>
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[N], const Q4Scale& s) {
  uint32_t word = 0;
  if (s.plain) {
    // float bits of 1.5 * 2^23 + code: the constant part of each is taken off the sum
    constexpr uint32_t kOnes = N == 8 ? 0x11111111u : N == 4 ? 0x1111u : 0u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      word += __float_as_uint(fminf(fmaf(x[i], s.inv, 48.f), 55.f) + (12582912.f - 40.f)) << (4 * i);
    return word - 0x4b400000u * kOnes;
  }
  // a scale that fp16 rounded (tiny or huge groups), no scale at all, NaN and infinities
  const float scale = __half2float(s.half);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = scale == 0.f ? 0.f : __fdiv_rn(x[i], scale);
    word |= (uint32_t)(min(max(__float2int_rn(y), -8), 7) + 8) << (4 * i);   // NaN converts to 0: code 8
  }
  return word;
}

// Which of the 16 rows from `first` on belong to 16 neighbouring rows that fill a tile: bit i for row first + i in `covered`;
// `leader`: the one that starts such a tile, or -1. Lane l < 16 gets slot[first + l].
struct Q4Window {
  uint32_t covered;
  int leader;
  long long slot;
};
__device__ __forceinline__ Q4Window q4_window(const long long* slots, long long first, long long T, long long num_slots) {
  const int lane = threadIdx.x & 31;
  // rows first - 16 + lane and first + 16 + lane; each knows whether the row after it is the next slot
  const long long i0 = first - 16 + lane, i1 = first + 16 + lane;
  const long long s0 = i0 >= 0 && i0 < T ? slots[i0] : -2, s1 = i1 < T ? slots[i1] : -2;
  long long n0 = __shfl_down_sync(0xffffffffu, s0, 1), n1 = __shfl_down_sync(0xffffffffu, s1, 1);
  const long long join = __shfl_sync(0xffffffffu, s1, 0);
  if (lane == 31) { n0 = join; n1 = -2; }
  const uint32_t c0 = __ballot_sync(0xffffffffu, s0 >= 0 && n0 == s0 + 1), c1 = __ballot_sync(0xffffffffu, s1 >= 0 && n1 == s1 + 1);
  const unsigned long long next = (unsigned long long)c1 << 32 | c0;           // bit j: row first - 16 + j
  Q4Window w;
  w.slot = __shfl_sync(0xffffffffu, s0, (lane & 15) + 16);
  const int into = (int)(w.slot & 15), bit = (lane & 15) + 16 - into;          // where the row's tile would start
  const bool in = w.slot >= 0 && w.slot < num_slots && (next >> bit & 0x7fffu) == 0x7fffu;
  w.covered = __ballot_sync(0xffffffffu, in) & 0xffffu;
  const uint32_t leads = __ballot_sync(0xffffffffu, in && into == 0) & 0xffffu;
  w.leader = leads != 0u ? __ffs(leads) - 1 : -1;
  return w;
}

// 8 neighbouring elements of a token's keys (pieces 0 .. hd / 8 - 1) or values (the rest); the four threads of a group are
// neighbours and all lanes of the warp take part.
template <bool BF16>
__device__ __forceinline__ void q4_put_piece(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint8_t* __restrict__ pool,
                                             long long t, long long slot, int h, int piece, bool live, int hkv, int hd, int tiles,
                                             long long k_stride, long long v_stride) {
  const int per = hd / 8, ng = hd / 32;
  const bool value = piece >= per;
  const int chunk = value ? piece - per : piece;
  uint4 u = make_uint4(0u, 0u, 0u, 0u);
  if (live) u = *reinterpret_cast<const uint4*>((value ? v + t * v_stride : k + t * k_stride) + h * hd + chunk * 8);
  float x[8];
  widen8<BF16>(u, x);
  float most = x[0], least = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    most = max_nan(most, x[e]);
    least = min_nan(least, x[e]);
  }
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
    least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, off));
  }
  if (!live) return;
  const Q4Scale s = q4_group(most, least);
  const uint32_t word = q4_codes(x, s);
  uint8_t* tile = pool + q4_tile_of(slot, h, hkv, tiles, q4_tile_bytes(hd));
  const int tok = (int)(slot & 15);
  if (value) {
    uint8_t* half = tile + 8 * hd;
    *reinterpret_cast<uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk)) = (uint16_t)word;
    *reinterpret_cast<uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk + 1)) = (uint16_t)(word >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(tile + q4_key_at(ng, tok, chunk)) = word;
  }
  if ((chunk & 3) == 0) reinterpret_cast<__half*>(tile + 16 * hd)[tok * 2 * ng + (value ? ng : 0) + (chunk >> 2)] = s.half;
}

template <bool BF16>
__global__ void __launch_bounds__(256)
kv_append_q4_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint8_t* __restrict__ pool,
                    const long long* __restrict__ slots, long long total, int hkv, int hd, int tiles, long long num_slots,
                    long long k_stride, long long v_stride) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per = hd / 4, piece = (int)(i % per);
  const long long th = i / per, t = th / hkv;
  const int h = (int)(th % hkv);
  const long long slot = i < total ? slots[t] : -1;
  q4_put_piece<BF16>(k, v, pool, t, slot, h, piece, slot >= 0 && slot < num_slots, hkv, hd, tiles, k_stride, v_stride);
}

__device__ __forceinline__ void q4_extremes2(uint32_t u, uint32_t& most, uint32_t& least, bool bf16) {
  if (bf16) {
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(most) : "r"(u));
    asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(least) : "r"(u));
  } else {
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(most) : "r"(u));
    asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(least) : "r"(u));
  }
}
template <bool BF16>
__device__ __forceinline__ float2 widen2(uint32_t u) {
  return BF16 ? unpack_bf16x2(u) : __half22float2(*reinterpret_cast<const __half2*>(&u));
}
// Scale of a group whose W registers are here, the rest in the lanes that differ in the bits OFF1 .. OFF2.
template <bool BF16, int W, int OFF1, int OFF2>
__device__ __forceinline__ Q4Scale q4_group_of(const uint32_t* u) {
  uint32_t most = u[0], least = u[0];
#pragma unroll
  for (int i = 1; i < W; ++i) q4_extremes2(u[i], most, least, BF16);
#pragma unroll
  for (int off = OFF1; off <= OFF2; off <<= 1) {
    const uint32_t a = __shfl_xor_sync(0xffffffffu, most, off), b = __shfl_xor_sync(0xffffffffu, least, off);
    uint32_t none = a;
    q4_extremes2(a, most, none, BF16);
    none = b;
    q4_extremes2(b, none, least, BF16);
  }
  const float2 a = widen2<BF16>(most), b = widen2<BF16>(least);
  return q4_group(max_nan(a.x, a.y), min_nan(b.x, b.y));
}

constexpr int kQ4RowWarps = 4;

// Grid (16-row windows, heads / 4): a warp has one head.
template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4RowWarps * 32)
kv_append_q4_tile_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint8_t* __restrict__ pool,
                         const long long* __restrict__ slots, long long T, int hkv, int tiles, long long num_slots,
                         long long k_stride, long long v_stride) {
  constexpr int HD = NG * 32;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int h = blockIdx.y * kQ4RowWarps + (threadIdx.x >> 5);
  if (h >= hkv) return;
  const long long first = (long long)blockIdx.x * 16;
  const Q4Window w = q4_window(slots, first, T, num_slots);
  if (w.leader >= 0) {
    const long long t0 = first + w.leader;
    uint8_t* tile = pool + q4_tile_of(__shfl_sync(0xffffffffu, w.slot, w.leader), h, hkv, tiles, 18 * HD);
    __half* scales = reinterpret_cast<__half*>(tile + 16 * HD);
    uint32_t word[2 * NG];
    // keys: tokens r, r + 8, elements 32 g + 8 c ..
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint16_t* from = k + (t0 + r + 8 * j) * k_stride + h * HD + c * 8;
      uint4 u[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) u[g] = *reinterpret_cast<const uint4*>(from + g * 32);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t x2[4] = {u[g].x, u[g].y, u[g].z, u[g].w};
        const Q4Scale s = q4_group_of<BF16, 4, 1, 2>(x2);
        float x[8];
        widen8<BF16>(u[g], x);
        word[j * NG + g] = q4_codes(x, s);
        if (c == 0) scales[(r + 8 * j) * 2 * NG + g] = s.half;
      }
    }
#pragma unroll
    for (int p = 0; p < NG / 2; ++p)
      *reinterpret_cast<uint4*>(tile + p * 512 + lane * 16) = make_uint4(word[4 * p], word[4 * p + 1], word[4 * p + 2], word[4 * p + 3]);
    // values: tokens 8 j + 2 c, + 1, elements 32 g + 4 r ..
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint2 u[2][NG];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint16_t* from = v + (t0 + 8 * j + 2 * c + e) * v_stride + h * HD + r * 4;
#pragma unroll
        for (int g = 0; g < NG; ++g) u[e][g] = *reinterpret_cast<const uint2*>(from + g * 32);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t both = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t x2[2] = {u[e][g].x, u[e][g].y};
          const Q4Scale s = q4_group_of<BF16, 2, 4, 16>(x2);
          const float2 lo = widen2<BF16>(x2[0]), hi = widen2<BF16>(x2[1]);
          const float x[4] = {lo.x, lo.y, hi.x, hi.y};
          both |= q4_codes(x, s) << (16 * e);
          if (r == 0) scales[(8 * j + 2 * c + e) * 2 * NG + NG + g] = s.half;
        }
        word[j * NG + g] = both;
      }
    }
#pragma unroll
    for (int p = 0; p < NG / 2; ++p)
      *reinterpret_cast<uint4*>(tile + 8 * HD + p * 512 + lane * 16) =
          make_uint4(word[4 * p], word[4 * p + 1], word[4 * p + 2], word[4 * p + 3]);
  }
  for (int i = 0; i < 16; ++i) {
    if (w.covered >> i & 1) continue;
    const long long slot = __shfl_sync(0xffffffffu, w.slot, i);
    if (slot < 0 || slot >= num_slots) continue;
#pragma unroll
    for (int p = 0; p < HD / 4; p += 32)
      q4_put_piece<BF16>(k, v, pool, first + i, slot, h, p + lane, p + lane < HD / 4, hkv, HD, tiles, k_stride, v_stride);
  }
}

// 8 elements from their codes.
template <bool BF16>
__device__ __forceinline__ uint32_t q4_value2(uint32_t a, uint32_t b, float scale) {
  // 2^23 + code as a float, less 2^23 + 8
  const float lo = (__uint_as_float(a | 0x4b000000u) - 8388616.f) * scale, hi = (__uint_as_float(b | 0x4b000000u) - 8388616.f) * scale;
  return BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
template <bool BF16>
__device__ __forceinline__ uint2 q4_values4(uint32_t codes, float scale) {
  return make_uint2(q4_value2<BF16>(codes & 15u, codes >> 4 & 15u, scale), q4_value2<BF16>(codes >> 8 & 15u, codes >> 12 & 15u, scale));
}

template <bool BF16>
__device__ __forceinline__ void q4_get_piece(const uint8_t* __restrict__ pool, uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                             long long t, long long slot, int h, int piece, bool live, int hkv, int hd, int tiles) {
  const int per = hd / 8, ng = hd / 32;
  const bool value = piece >= per;
  const int chunk = value ? piece - per : piece;
  uint4 out = make_uint4(0u, 0u, 0u, 0u);
  if (live) {
    const uint8_t* tile = pool + q4_tile_of(slot, h, hkv, tiles, q4_tile_bytes(hd));
    const int tok = (int)(slot & 15);
    uint32_t word;
    if (value) {
      const uint8_t* half = tile + 8 * hd;
      word = *reinterpret_cast<const uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk)) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk + 1)) << 16;
    } else {
      word = *reinterpret_cast<const uint32_t*>(tile + q4_key_at(ng, tok, chunk));
    }
    const float scale = __half2float(reinterpret_cast<const __half*>(tile + 16 * hd)[tok * 2 * ng + (value ? ng : 0) + (chunk >> 2)]);
    const uint2 a = q4_values4<BF16>(word & 0xffffu, scale), b = q4_values4<BF16>(word >> 16, scale);
    out = make_uint4(a.x, a.y, b.x, b.y);
  }
  *reinterpret_cast<uint4*>((value ? v : k) + (t * hkv + h) * hd + chunk * 8) = out;
}

template <bool BF16>
__global__ void __launch_bounds__(256)
kv_read_q4_kernel(const uint8_t* __restrict__ pool, const long long* __restrict__ slots, uint16_t* __restrict__ k,
                  uint16_t* __restrict__ v, long long total, int hkv, int hd, int tiles, long long num_slots) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int per = hd / 4, piece = (int)(i % per);
  const long long th = i / per, t = th / hkv;
  const long long slot = slots[t];
  q4_get_piece<BF16>(pool, k, v, t, slot, (int)(th % hkv), piece, slot >= 0 && slot < num_slots, hkv, hd, tiles);
}

template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4RowWarps * 32)
kv_read_q4_tile_kernel(const uint8_t* __restrict__ pool, const long long* __restrict__ slots, uint16_t* __restrict__ k,
                       uint16_t* __restrict__ v, long long T, int hkv, int tiles, long long num_slots) {
  constexpr int HD = NG * 32;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int h = blockIdx.y * kQ4RowWarps + (threadIdx.x >> 5);
  if (h >= hkv) return;
  const long long first = (long long)blockIdx.x * 16;
  const Q4Window w = q4_window(slots, first, T, num_slots);
  if (w.leader >= 0) {
    const long long t0 = first + w.leader, pitch = (long long)hkv * HD;
    const uint8_t* tile = pool + q4_tile_of(__shfl_sync(0xffffffffu, w.slot, w.leader), h, hkv, tiles, 18 * HD);
    const __half* scales = reinterpret_cast<const __half*>(tile + 16 * HD);
    uint32_t kw[2 * NG], vw[2 * NG];
#pragma unroll
    for (int p = 0; p < NG / 2; ++p) {
      const uint4 a = *reinterpret_cast<const uint4*>(tile + p * 512 + lane * 16);
      const uint4 b = *reinterpret_cast<const uint4*>(tile + 8 * HD + p * 512 + lane * 16);
      kw[4 * p] = a.x; kw[4 * p + 1] = a.y; kw[4 * p + 2] = a.z; kw[4 * p + 3] = a.w;
      vw[4 * p] = b.x; vw[4 * p + 1] = b.y; vw[4 * p + 2] = b.z; vw[4 * p + 3] = b.w;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint16_t* to = k + (t0 + r + 8 * j) * pitch + h * HD + c * 8;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float scale = __half2float(scales[(r + 8 * j) * 2 * NG + g]);
        const uint32_t word = kw[j * NG + g];
        const uint2 a = q4_values4<BF16>(word & 0xffffu, scale), b = q4_values4<BF16>(word >> 16, scale);
        *reinterpret_cast<uint4*>(to + g * 32) = make_uint4(a.x, a.y, b.x, b.y);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tok = 8 * j + 2 * c + e;
        uint16_t* out = v + (t0 + tok) * pitch + h * HD + r * 4;
#pragma unroll
        for (int g = 0; g < NG; ++g)
          *reinterpret_cast<uint2*>(out + g * 32) =
              q4_values4<BF16>(e ? vw[j * NG + g] >> 16 : vw[j * NG + g] & 0xffffu, __half2float(scales[tok * 2 * NG + NG + g]));
      }
    }
  }
  for (int i = 0; i < 16 && first + i < T; ++i) {
    if (w.covered >> i & 1) continue;
    const long long slot = __shfl_sync(0xffffffffu, w.slot, i);
    for (int p = lane; p < HD / 4; p += 32)
      q4_get_piece<BF16>(pool, k, v, first + i, slot, h, p, slot >= 0 && slot < num_slots, hkv, HD, tiles);
  }
}

// Rows from which on the kernels by tiles take a call. Few rows are a decode step's, no two of them in a tile, or a prompt that
// one launch of either kind is too short for.
constexpr long long kQ4TileRows = 512;

}  // namespace icb

using namespace icb;

#define ICB_Q4_SIZES(RUN) \
  switch (hd / 64) { \
    case 1: RUN(2) break; \
    case 2: RUN(4) break; \
    case 3: RUN(6) break; \
    case 4: RUN(8) break; \
    default: return -3; \
  }

// k, v: [T, hkv * hd] 16-bit rows of pitch k_stride / v_stride (16-byte aligned); pool: num_slots / (16 * tiles) pages of
// [hkv][tiles] tiles; a row whose slot is negative or outside the pool is left out. hd 64, 128, 192 or 256.
ICB_API int icb_kv_append_q4(const void* k, const void* v, void* pool, const long long* slots, long long T, int hkv, int hd,
                             int tiles, long long num_slots, long long k_stride, long long v_stride, int dtype,
                             void* stream) {
  if (T <= 0) return 0;
  if (hkv < 1 || hd % 64 || hd < 64 || hd > 256 || tiles < 1 || k_stride % 8 || v_stride % 8) return -2;
  if (dtype != kBF16 && dtype != kF16) return -4;
  auto K = reinterpret_cast<const uint16_t*>(k), V = reinterpret_cast<const uint16_t*>(v);
  auto p = reinterpret_cast<uint8_t*>(pool);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (T >= kQ4TileRows) {
    const dim3 grid((unsigned)((T + 15) / 16), (hkv + kQ4RowWarps - 1) / kQ4RowWarps);
    if ((T + 15) / 16 > 0x7fffffffLL || grid.y > 65535) return -3;
#define ICB_RUN(NG_) \
    if (dtype == kBF16) kv_append_q4_tile_kernel<NG_, true><<<grid, kQ4RowWarps * 32, 0, st>>>(K, V, p, slots, T, hkv, tiles, num_slots, k_stride, v_stride); \
    else kv_append_q4_tile_kernel<NG_, false><<<grid, kQ4RowWarps * 32, 0, st>>>(K, V, p, slots, T, hkv, tiles, num_slots, k_stride, v_stride);
    ICB_Q4_SIZES(ICB_RUN)
#undef ICB_RUN
  } else {
    const long long total = T * hkv * (hd / 4), blocks = (total + 255) / 256;
    if (blocks > 0x7fffffffLL) return -3;
    if (dtype == kBF16) kv_append_q4_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(K, V, p, slots, total, hkv, hd, tiles, num_slots, k_stride, v_stride);
    else kv_append_q4_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(K, V, p, slots, total, hkv, hd, tiles, num_slots, k_stride, v_stride);
  }
  return check_launch("kv_append_q4");
}

// The rows `slots` of the pool as 16-bit k, v [T, hkv * hd]; zeros for a slot outside the pool.
ICB_API int icb_kv_read_q4(const void* pool, const long long* slots, void* k, void* v, long long T, int hkv, int hd,
                           int tiles, long long num_slots, int dtype, void* stream) {
  if (T <= 0) return 0;
  if (hkv < 1 || hd % 64 || hd < 64 || hd > 256 || tiles < 1) return -2;
  if (dtype != kBF16 && dtype != kF16) return -4;
  auto K = reinterpret_cast<uint16_t*>(k), V = reinterpret_cast<uint16_t*>(v);
  auto p = reinterpret_cast<const uint8_t*>(pool);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (T >= kQ4TileRows) {
    const dim3 grid((unsigned)((T + 15) / 16), (hkv + kQ4RowWarps - 1) / kQ4RowWarps);
    if ((T + 15) / 16 > 0x7fffffffLL || grid.y > 65535) return -3;
#define ICB_RUN(NG_) \
    if (dtype == kBF16) kv_read_q4_tile_kernel<NG_, true><<<grid, kQ4RowWarps * 32, 0, st>>>(p, slots, K, V, T, hkv, tiles, num_slots); \
    else kv_read_q4_tile_kernel<NG_, false><<<grid, kQ4RowWarps * 32, 0, st>>>(p, slots, K, V, T, hkv, tiles, num_slots);
    ICB_Q4_SIZES(ICB_RUN)
#undef ICB_RUN
  } else {
    const long long total = T * hkv * (hd / 4), blocks = (total + 255) / 256;
    if (blocks > 0x7fffffffLL) return -3;
    if (dtype == kBF16) kv_read_q4_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(p, slots, K, V, total, hkv, hd, tiles, num_slots);
    else kv_read_q4_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(p, slots, K, V, total, hkv, hd, tiles, num_slots);
  }
  return check_launch("kv_read_q4");
}
