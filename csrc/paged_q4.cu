// Rows of the 4-bit paged key / value cache (format: q4.cuh): quantise and write, read back.
//
// Quantisation of a group of 32 elements: scale = m / -8 rounded to fp16, m the element of largest magnitude (the largest
// if the smallest is as far from zero), so that m itself is code 0 and the other end of the range reaches code 15;
// n = clamp(round(x / scale), -8, 7) + 8, ties to even.
//
// Rounding without a division: x and scale have at most 11 significant bits, so x / scale is either a tie k + 1/2 or differs
// from one by at least 2^-15 of its value, 2^-16 or more. y = x * (1 / scale) with a reciprocal within 2^-23 is off by at most
// 2^-20 (|y| <= 8), and fma(x, 1 / scale, 48) rounds it to a multiple of 2^-18: ties come out as ties, everything else stays on
// its side of them. Adding 1.5 * 2^23 - 40 then rounds to an integer, ties to even, whose low bits are the code.
//
// Two forms of each direction: one thread per 8 elements of a row, for few rows; and four warps per tile of 16 rows and head, in
// the order of the tile's lanes, so that all 18 hd bytes of the tile leave or arrive in 512-byte pieces (a row by itself touches
// all of a tile's value sectors, two bytes in each). Rows that do not fill a tile go one by one. 32768 rows of 8 heads of 128:
// append 41 us from a cold cache, 0.64 of the copy bandwidth, held by instruction issue (0.68 of the slots: eleven instructions an
// element, half of them conversion and rounding); read 32 us, 0.83, held by its writes. One warp per tile took 61 and 39 us.
#include <string.h>

#include "host_common.h"
#include "launch_behind.cuh"
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

struct Q4Scale {
  __half half;
  float inv;                    // its reciprocal, within 2^-23
  bool plain;                   // the largest element is -8 scales exactly: no code can be below 0
};
// From the extremes of a group; a NaN among the elements makes both NaN.
__device__ __forceinline__ Q4Scale q4_group(float most, float least) {
  const float m = most >= -least ? most : least;
  Q4Scale s;
  s.half = __float2half_rn(fmaf(m, -0.125f, 0.f));            // the sum has no negative zero
  const float scale = __half2float(s.half);
  s.plain = scale * -8.f == m && fabsf(m) <= 524032.f;      // an infinity is not
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.inv) : "f"(scale));
  if (scale == 0.f) s.inv = 0.f;
  if (!s.plain) {                                             // rounded (tiny groups), too large for fp16, NaN
    float x = m * -0.125f;
    if (x > 65504.f) x = 65504.f;
    if (x < -65504.f) x = -65504.f;
    s.half = __float2half_rn(x);
    if (__half2float(s.half) == 0.f) s.half = __ushort_as_half(0);
  }
  return s;
}

__device__ __forceinline__ unsigned long long bits2(const float2& a) { return *reinterpret_cast<const unsigned long long*>(&a); }
__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return *reinterpret_cast<float2*>(&d);
}

// N codes (at most 8) of a plain group, lowest nibble first.
template <int N>
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[N], float inv) {
  // float bits of 1.5 * 2^23 + code: the constant part of each is taken off the sum
  constexpr uint32_t kOnes = N == 8 ? 0x11111111u : N == 4 ? 0x1111u : 0u;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 y = ffma2(make_float2(x[i], x[i + 1]), make_float2(inv, inv), make_float2(48.f, 48.f));
    y = fadd2(make_float2(fminf(y.x, 55.f), fminf(y.y, 55.f)), make_float2(12582912.f - 40.f, 12582912.f - 40.f));
    word += (__float_as_uint(y.x) << (4 * i)) + (__float_as_uint(y.y) << (4 * i + 4));
  }
  return word - 0x4b400000u * kOnes;
}
// Of any group: a scale that fp16 rounded (tiny or huge groups), no scale at all, NaN and infinities.
__device__ __noinline__ uint32_t q4_codes_any(float scale, float x0, float x1, float x2, float x3, float x4, float x5, float x6,
                                              float x7) {
  const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
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

// A piece: 8 neighbouring elements of a token's keys (pieces 0 .. hd / 8 - 1) or values (the rest). The four threads of a group
// are neighbours and all lanes of the warp take part.
__device__ __forceinline__ const uint16_t* q4_piece_of(const uint16_t* k, const uint16_t* v, long long t, int h, int piece, int hd,
                                                       long long k_stride, long long v_stride) {
  const int per = hd / 8;
  return (piece >= per ? v + t * v_stride + (piece - per) * 8 : k + t * k_stride + piece * 8) + h * hd;
}
// Out of line where a kernel has it beside other work: what runs once a launch costs the fetching of its instructions.
template <bool BF16>
__device__ __noinline__ void q4_put_piece(const uint4& u, uint8_t* __restrict__ pool, long long slot, int h, int piece, bool live,
                                             int hkv, int hd, int tiles) {
  const int per = hd / 8, ng = hd / 32;
  const bool value = piece >= per;
  const int chunk = value ? piece - per : piece;
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
  const uint32_t word = s.plain ? q4_codes(x, s.inv)
                                : q4_codes_any(__half2float(s.half), x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
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
  wait_for_previous();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per = hd / 4, piece = (int)(i % per);
  const long long th = i / per, t = th / hkv;
  const int h = (int)(th % hkv);
  const long long slot = i < total ? slots[t] : -1;
  const bool live = slot >= 0 && slot < num_slots;
  uint4 u = make_uint4(0u, 0u, 0u, 0u);
  if (live) u = *reinterpret_cast<const uint4*>(q4_piece_of(k, v, t, h, piece, hd, k_stride, v_stride));
  q4_put_piece<BF16>(u, pool, slot, h, piece, live, hkv, hd, tiles);
}

template <bool BF16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  if (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t d;
  if (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16>
__device__ __forceinline__ float2 widen2(uint32_t u) {
  return BF16 ? unpack_bf16x2(u) : __half22float2(*reinterpret_cast<const __half2*>(&u));
}
// (largest element, largest negated element) of W registers.
template <bool BF16, int W>
__device__ __forceinline__ uint32_t q4_extremes(const uint32_t* u) {
  uint32_t most = u[0], least = u[0];
#pragma unroll
  for (int i = 1; i < W; ++i) {
    most = max2<BF16>(most, u[i]);
    least = min2<BF16>(least, u[i]);
  }
  least ^= 0x80008000u;
  return max2<BF16>(__byte_perm(most, least, 0x5410), __byte_perm(most, least, 0x7632));
}
// N groups' extremes, each spread over the lanes that differ in the bits OFF, OFF / 2 .. LAST: halving the groups at each step
// while their number is even leaves q4_owned() of them with every lane, all lanes' work on scales being different.
__host__ __device__ constexpr int q4_owned(int n, int steps) { return steps == 0 || n % 2 ? n : q4_owned(n / 2, steps - 1); }
template <bool BF16, int N, int OFF, int LAST>
__device__ __forceinline__ void q4_gather(uint32_t* m) {
  constexpr int KEEP = N % 2 ? N : N / 2;
  const bool up = (threadIdx.x & OFF) != 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const uint32_t send = N % 2 || up ? m[i] : m[i + N - KEEP], keep = N % 2 || !up ? m[i] : m[i + N - KEEP];
    m[i] = max2<BF16>(keep, __shfl_xor_sync(0xffffffffu, send, OFF));
  }
  if constexpr (OFF > LAST) q4_gather<BF16, KEEP, OFF / 2, LAST>(m);
}

// NG fp16 scales at once (p aligned to them).
template <int NG>
__device__ __forceinline__ void get_scales(const __half* p, __half (&s)[NG]) {
  if (NG == 8) *reinterpret_cast<uint4*>(s) = *reinterpret_cast<const uint4*>(p);
  else if (NG == 4) *reinterpret_cast<uint2*>(s) = *reinterpret_cast<const uint2*>(p);
  else {
#pragma unroll
    for (int i = 0; i < NG; i += 2) *reinterpret_cast<uint32_t*>(s + i) = *reinterpret_cast<const uint32_t*>(p + i);
  }
}

// The words i0 .. i0 + NG - 1 of this lane in one half of a tile.
template <int NG>
__device__ __forceinline__ void put_words(uint8_t* half, int i0, const uint32_t (&w)[NG]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NG; i += (NG % 4 == 0 ? 4 : 2)) {
    uint8_t* to = half + q4_word_at(i0 + i, lane);
    if (NG % 4 == 0) *reinterpret_cast<uint4*>(to) = make_uint4(w[i], w[i + 1], w[(i + 2) % NG], w[(i + 3) % NG]);
    else *reinterpret_cast<uint2*>(to) = make_uint2(w[i], w[i + 1]);
  }
}
template <int NG>
__device__ __forceinline__ void get_words(const uint8_t* half, int i0, uint32_t (&w)[NG]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NG; i += (NG % 4 == 0 ? 4 : 2)) {
    const uint8_t* from = half + q4_word_at(i0 + i, lane);
    if (NG % 4 == 0) {
      const uint4 u = *reinterpret_cast<const uint4*>(from);
      w[i] = u.x; w[i + 1] = u.y; w[(i + 2) % NG] = u.z; w[(i + 3) % NG] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(from);
      w[i] = u.x; w[i + 1] = u.y;
    }
  }
}

constexpr int kQ4RowWarps = 4;

// Grid (16-row windows, runs of heads). A tile's work is shared by four warps: keys and values, first and second 8 tokens.
template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4RowWarps * 32)
kv_append_q4_tile_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint8_t* __restrict__ pool,
                         const long long* __restrict__ slots, long long T, int hkv, int tiles, long long num_slots,
                         long long k_stride, long long v_stride, int per) {
  constexpr int HD = NG * 32, PIECES = (HD / 4 + 31) / 32, DEPTH = 4;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, warp = threadIdx.x >> 5, j = warp & 1;
  const int h0 = blockIdx.y * per, h1 = min(hkv, h0 + per);
  const long long first = (long long)blockIdx.x * 16;
  wait_for_previous();
  const Q4Window w = q4_window(slots, first, T, num_slots);
  const uint32_t valid = __ballot_sync(0xffffffffu, lane < 16 && w.slot >= 0 && w.slot < num_slots);
  const uint32_t single = valid & ~w.covered & (0x1111u << warp);
  const long long t0 = first + w.leader, slot0 = __shfl_sync(0xffffffffu, w.slot, w.leader & 15);
  const bool keys = warp < 2;
  const int tok = 8 * j + (keys ? r : 2 * c);    // the lane's token, for values the first of two
  uint8_t* tile = pool + q4_tile_of(slot0, h0, hkv, tiles, 18 * HD);
  const uint16_t* from = keys ? k + (t0 + tok) * k_stride + h0 * HD + c * 8 : v + (t0 + tok) * v_stride + h0 * HD + r * 4;
#pragma unroll 1
  for (int h = h0; h < h1; ++h, tile += (size_t)tiles * 18 * HD, from += HD) {
    // rows that go one by one: bit i for row row0 + i, whose slot lane i has; pieces p0 to p1 of them
    long long row0 = first, slot = w.slot;
    uint32_t left = 0;
    int p0 = 0, p1 = HD / 4;
    if (w.leader >= 0) {
      __half* scales = reinterpret_cast<__half*>(tile + 16 * HD);
      uint32_t word[NG];
      bool plain = true;
      if (keys) {                                // elements 32 g + 8 c .. of a token
        constexpr int OWN = q4_owned(NG, 2), SHIFT = NG / OWN == 4 ? 0 : 1;
        uint4 u[NG];
        uint32_t m[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) u[g] = *reinterpret_cast<const uint4*>(from + g * 32);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint32_t x2[4] = {u[g].x, u[g].y, u[g].z, u[g].w};
          m[g] = q4_extremes<BF16, 4>(x2);
        }
        q4_gather<BF16, NG, 2, 1>(m);
        float inv[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const float2 x = widen2<BF16>(m[i]);
          const Q4Scale s = q4_group(x.x, -x.y);
          inv[i] = s.inv;
          plain &= s.plain;
          scales[tok * 2 * NG + (c >> SHIFT) * OWN + i] = s.half;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float x[8];
          widen8<BF16>(u[g], x);
          word[g] = q4_codes(x, __shfl_sync(0xffffffffu, inv[g % OWN], 4 * r + (g / OWN << SHIFT)));
        }
        put_words<NG>(tile, j * NG, word);
        p1 = HD / 8;
      } else {                                   // elements 32 g + 4 r .. of two tokens
        constexpr int OWN = q4_owned(2 * NG, 3), SHIFT = 2 * NG / OWN == 8 ? 0 : 1;
        uint2 u[2][NG];
        uint32_t m[2 * NG];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int g = 0; g < NG; ++g) u[e][g] = *reinterpret_cast<const uint2*>(from + e * v_stride + g * 32);
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) {
          const uint32_t x2[2] = {u[i / NG][i % NG].x, u[i / NG][i % NG].y};
          m[i] = q4_extremes<BF16, 2>(x2);
        }
        q4_gather<BF16, 2 * NG, 16, 4>(m);
        float inv[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const float2 x = widen2<BF16>(m[i]);
          const Q4Scale s = q4_group(x.x, -x.y);
          inv[i] = s.inv;
          plain &= s.plain;
          const int which = (r >> SHIFT) * OWN + i, e = which >= NG;
          scales[(tok + e) * 2 * NG + NG + which - e * NG] = s.half;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) word[g] = 0;
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) {
          const uint2& t = u[i / NG][i % NG];
          const float2 lo = widen2<BF16>(t.x), hi = widen2<BF16>(t.y);
          const float x[4] = {lo.x, lo.y, hi.x, hi.y};
          word[i % NG] |= q4_codes(x, __shfl_sync(0xffffffffu, inv[i % OWN], 4 * (i / OWN << SHIFT) + c)) << (16 * (i / NG));
        }
        put_words<NG>(tile + 8 * HD, j * NG, word);
        p0 = HD / 8;
      }
      if (!__all_sync(0xffffffffu, plain)) {     // a group needs the long way: the warp's part takes it, over what it wrote
        __syncwarp();
        row0 = t0;
        slot = slot0 + (lane & 15);
        left = 0xffu << (8 * j);
      }
    }
    if ((left | single) == 0u) continue;
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {       // the warp's part once more, then its share of the rows that fill no tile
      while (left != 0u) {
        uint4 u[DEPTH][PIECES];                  // some rows at a time, so that their loads share a wait
        uint32_t rest = left;
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
          const int row = __ffs(rest) - 1;
#pragma unroll
          for (int p = 0; p < PIECES; ++p) {
            const int piece = p0 + p * 32 + lane;
            u[i][p] = make_uint4(0u, 0u, 0u, 0u);
            if (row >= 0 && piece < p1)
              u[i][p] = *reinterpret_cast<const uint4*>(q4_piece_of(k, v, row0 + row, h, piece, HD, k_stride, v_stride));
          }
          rest &= rest - 1;
        }
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
          if (left == 0u) break;
          const long long at = __shfl_sync(0xffffffffu, slot, __ffs(left) - 1);
#pragma unroll
          for (int p = 0; p < PIECES; ++p) {
            const int piece = p0 + p * 32 + lane;
            q4_put_piece<BF16>(u[i][p], pool, at, h, piece, piece < p1, hkv, HD, tiles);
          }
          left &= left - 1;
        }
      }
      if (turn == 1) break;
      row0 = first;
      slot = w.slot;
      p0 = 0;
      p1 = HD / 4;
      left = single;
    }
  }
}

// 4 elements from their codes: a nibble at the bottom of the upper half of 0x43000000 is the float 128 + code.
template <bool BF16>
__device__ __forceinline__ uint32_t q4_value2(uint32_t a, uint32_t b, float scale) {
  const float lo = __uint_as_float((a & 0xf0000u) | 0x43000000u), hi = __uint_as_float((b & 0xf0000u) | 0x43000000u);
  const float2 n = fadd2(make_float2(lo, hi), make_float2(-136.f, -136.f));
  const float2 x = fmul2(n, make_float2(scale, scale));
  return BF16 ? pack_bf16x2(x.x, x.y) : pack_f16x2(x.x, x.y);
}
template <bool BF16, int AT>                     // the codes at bits AT .. AT + 15
__device__ __forceinline__ uint2 q4_values4(uint32_t word, float scale) {
  return AT == 0 ? make_uint2(q4_value2<BF16>(word << 16, word << 12, scale), q4_value2<BF16>(word << 8, word << 4, scale))
                 : make_uint2(q4_value2<BF16>(word, word >> 4, scale), q4_value2<BF16>(word >> 8, word >> 12, scale));
}

struct Q4Piece {
  uint32_t word;
  __half scale;
};
__device__ __forceinline__ Q4Piece q4_get_piece(const uint8_t* __restrict__ pool, long long slot, int h, int piece, bool live, int hkv,
                                                int hd, int tiles) {
  Q4Piece x{0x88888888u, __ushort_as_half(0)};    // zeros
  if (!live) return x;
  const int per = hd / 8, ng = hd / 32;
  const bool value = piece >= per;
  const int chunk = value ? piece - per : piece, tok = (int)(slot & 15);
  const uint8_t* tile = pool + q4_tile_of(slot, h, hkv, tiles, q4_tile_bytes(hd));
  if (value) {
    const uint8_t* half = tile + 8 * hd;
    x.word = *reinterpret_cast<const uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk)) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk + 1)) << 16;
  } else {
    x.word = *reinterpret_cast<const uint32_t*>(tile + q4_key_at(ng, tok, chunk));
  }
  x.scale = reinterpret_cast<const __half*>(tile + 16 * hd)[tok * 2 * ng + (value ? ng : 0) + (chunk >> 2)];
  return x;
}
template <bool BF16>
__device__ __forceinline__ void q4_write_piece(const Q4Piece& x, uint16_t* __restrict__ k, uint16_t* __restrict__ v, long long t,
                                               int h, int piece, int hkv, int hd) {
  const int per = hd / 8;
  const float scale = __half2float(x.scale);
  const uint2 a = q4_values4<BF16, 0>(x.word, scale), b = q4_values4<BF16, 16>(x.word, scale);
  uint16_t* to = (piece >= per ? v + (piece - per) * 8 : k + piece * 8) + (t * hkv + h) * hd;
  *reinterpret_cast<uint4*>(to) = make_uint4(a.x, a.y, b.x, b.y);
}

template <bool BF16>
__global__ void __launch_bounds__(256)
kv_read_q4_kernel(const uint8_t* __restrict__ pool, const long long* __restrict__ slots, uint16_t* __restrict__ k,
                  uint16_t* __restrict__ v, long long total, int hkv, int hd, int tiles, long long num_slots) {
  wait_for_previous();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int per = hd / 4, piece = (int)(i % per);
  const long long th = i / per, t = th / hkv;
  const long long slot = slots[t];
  const int h = (int)(th % hkv);
  const Q4Piece x = q4_get_piece(pool, slot, h, piece, slot >= 0 && slot < num_slots, hkv, hd, tiles);
  q4_write_piece<BF16>(x, k, v, t, h, piece, hkv, hd);
}

template <int NG, bool BF16>
__global__ void __launch_bounds__(kQ4RowWarps * 32)
kv_read_q4_tile_kernel(const uint8_t* __restrict__ pool, const long long* __restrict__ slots, uint16_t* __restrict__ k,
                       uint16_t* __restrict__ v, long long T, int hkv, int tiles, long long num_slots, int per) {
  constexpr int HD = NG * 32, PIECES = (HD / 4 + 31) / 32, DEPTH = 4;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, warp = threadIdx.x >> 5, j = warp & 1;
  const int h0 = blockIdx.y * per, h1 = min(hkv, h0 + per);
  const long long first = (long long)blockIdx.x * 16, pitch = (long long)hkv * HD;
  wait_for_previous();
  const Q4Window w = q4_window(slots, first, T, num_slots);
  // this warp's share of the rows that fill no tile
  const uint32_t single = ~w.covered & (first + 16 <= T ? 0xffffu : (1u << (T - first)) - 1u) & (0x1111u << warp);
  const long long t0 = first + w.leader, slot0 = __shfl_sync(0xffffffffu, w.slot, w.leader & 15);
  const bool keys = warp < 2;
  const int tok = 8 * j + (keys ? r : 2 * c);
  const uint8_t* tile = pool + q4_tile_of(slot0, h0, hkv, tiles, 18 * HD);
  uint16_t* to = keys ? k + (t0 + tok) * pitch + h0 * HD + c * 8 : v + (t0 + tok) * pitch + h0 * HD + r * 4;
#pragma unroll 1
  for (int h = h0; h < h1; ++h, tile += (size_t)tiles * 18 * HD, to += HD) {
    if (w.leader >= 0) {
      const __half* scales = reinterpret_cast<const __half*>(tile + 16 * HD) + tok * 2 * NG;
      uint32_t word[NG];
      if (keys) {                                // elements 32 g + 8 c .. of a token
        __align__(16) __half row[NG];
        get_words<NG>(tile, j * NG, word);
        get_scales<NG>(scales, row);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float scale = __half2float(row[g]);
          const uint2 a = q4_values4<BF16, 0>(word[g], scale), b = q4_values4<BF16, 16>(word[g], scale);
          *reinterpret_cast<uint4*>(to + g * 32) = make_uint4(a.x, a.y, b.x, b.y);
        }
      } else {                                   // elements 32 g + 4 r .. of two tokens
        __align__(16) __half row[2][NG];
        get_words<NG>(tile + 8 * HD, j * NG, word);
#pragma unroll
        for (int e = 0; e < 2; ++e) get_scales<NG>(scales + e * 2 * NG + NG, row[e]);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          *reinterpret_cast<uint2*>(to + g * 32) = q4_values4<BF16, 0>(word[g], __half2float(row[0][g]));
          *reinterpret_cast<uint2*>(to + pitch + g * 32) = q4_values4<BF16, 16>(word[g], __half2float(row[1][g]));
        }
      }
    }
    uint32_t left = single;
    while (left != 0u) {
      Q4Piece x[DEPTH][PIECES];                  // some rows at a time, so that their loads share a wait
      uint32_t rest = left;
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        const int row = __ffs(rest) - 1;
        const long long slot = __shfl_sync(0xffffffffu, w.slot, max(row, 0));
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          const int piece = p * 32 + lane;
          const bool there = row >= 0 && piece < HD / 4 && slot >= 0 && slot < num_slots;
          x[i][p] = q4_get_piece(pool, slot, h, piece, there, hkv, HD, tiles);
        }
        rest &= rest - 1;
      }
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        if (left == 0u) break;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
          if (p * 32 + lane < HD / 4) q4_write_piece<BF16>(x[i][p], k, v, first + __ffs(left) - 1, h, p * 32 + lane, hkv, HD);
        left &= left - 1;
      }
    }
  }
}

// Elements of the keys from which on the kernels by tiles take a call. What pays depends on the slots, which are on the device: rows
// in order gain by tiles, rows that lie in a tile each (a decode step) lose. By rows / by tiles, us, from graphs: append, 8 heads of
// 128, in order, 512 rows 3.1 / 2.2, 2048 rows (the threshold) 7.8 / 3.7, 8192 rows 27 / 12, 32768 rows 100 / 34; scattered,
// 512 rows 3.1 / 5.1, 2048 rows 8.6 / 10.6, 8192 rows 27 / 35; 1 head of 256, 8192 rows (the threshold) in order 7.1 / 3.9,
// scattered 7.9 / 12.9. Read, 8 heads of 128, in order, 2048 rows 6.3 / 3.1, scattered 7.4 / 7.4; 1 head of 256, 8192 rows 5.6
// / 3.1 and 6.3 / 6.2. So the threshold lies above the decode steps but for the largest: 512 sequences of 32 heads of 128 are
// on it, 10.7 us instead of 8.6.
constexpr long long kQ4TileElements = 1LL << 21;

// Heads that a block goes through one after the other, so that its look at the slots serves them all; blocks stay enough for 32
// to an SM, since one with rows that fill no tile takes longer than others: 16 sequences of up to 4000 rows, 8 heads of 128, append
// 40.9 us with 16 to an SM, 36.4 with 32, 42.1 with 64; read 39.6, 35.3, 38.6.
static int q4_heads_per_block(long long T, int hkv) {
  const long long all = (T + 15) / 16 * hkv, per = all / (32LL * num_sms());
  return per < 1 ? 1 : per < hkv ? (int)per : hkv;
}

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

// The arguments of both entry points come as one record (a caller through ctypes spends a third of the time on it).
//   k, v: [rows, hkv * hd] 16-bit rows of pitch k_stride / v_stride (16-byte aligned; read: contiguous); pool: num_slots /
//   (16 * tiles) pages of [hkv][tiles] tiles; slots: int64 [rows]. hd 64, 128, 192 or 256.
struct Q4RowsCall {
  uint16_t *k, *v;
  uint8_t* pool;
  const long long* slots;
  long long rows, hkv, hd, tiles, num_slots, k_stride, v_stride, dtype;
};
static int q4_rows_call(Q4RowsCall& c, const void* record) {
  memcpy(&c, record, sizeof(c));
  if (c.hkv < 1 || c.hkv > 0x7fffffffLL || c.tiles < 1 || c.tiles > 0x7fffffffLL || c.k_stride % 8 || c.v_stride % 8) return -2;
  if (c.hd % 64 || c.hd < 64 || c.hd > 256) return -3;
  return c.dtype == kBF16 || c.dtype == kF16 ? 0 : -4;
}

// Quantises rows into the pool; a row whose slot is negative or outside the pool is left out.
ICB_API int icb_kv_append_q4(const void* record, void* stream) {
  Q4RowsCall c;
  const int bad = q4_rows_call(c, record);
  if (bad) return bad;
  if (c.rows <= 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int hkv = (int)c.hkv, hd = (int)c.hd, tiles = (int)c.tiles;
  if (c.rows * hkv * hd >= kQ4TileElements) {
    const int per = q4_heads_per_block(c.rows, hkv);
    const dim3 grid((unsigned)((c.rows + 15) / 16), (hkv + per - 1) / per);
    if ((c.rows + 15) / 16 > 0x7fffffffLL || grid.y > 65535) return -3;
#define ICB_RUN(NG_) { \
      auto kernel = c.dtype == kBF16 ? kv_append_q4_tile_kernel<NG_, true> : kv_append_q4_tile_kernel<NG_, false>; \
      return launch_behind("kv_append_q4", kernel, grid, kQ4RowWarps * 32, 0, st, c.k, c.v, c.pool, c.slots, c.rows, hkv, \
                           tiles, c.num_slots, c.k_stride, c.v_stride, per); \
    }
    ICB_Q4_SIZES(ICB_RUN)
#undef ICB_RUN
  } else {
    const long long total = c.rows * hkv * (hd / 4), blocks = (total + 255) / 256;
    if (blocks > 0x7fffffffLL) return -3;
    auto kernel = c.dtype == kBF16 ? kv_append_q4_kernel<true> : kv_append_q4_kernel<false>;
    return launch_behind("kv_append_q4", kernel, (unsigned)blocks, 256, 0, st, c.k, c.v, c.pool, c.slots, total, hkv, hd, tiles,
                         c.num_slots, c.k_stride, c.v_stride);
  }
}

// Rows of the pool in 16 bits; zeros for a slot outside the pool.
ICB_API int icb_kv_read_q4(const void* record, void* stream) {
  Q4RowsCall c;
  const int bad = q4_rows_call(c, record);
  if (bad) return bad;
  if (c.rows <= 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int hkv = (int)c.hkv, hd = (int)c.hd, tiles = (int)c.tiles;
  if (c.rows * hkv * hd >= kQ4TileElements) {
    const int per = q4_heads_per_block(c.rows, hkv);
    const dim3 grid((unsigned)((c.rows + 15) / 16), (hkv + per - 1) / per);
    if ((c.rows + 15) / 16 > 0x7fffffffLL || grid.y > 65535) return -3;
#define ICB_RUN(NG_) { \
      auto kernel = c.dtype == kBF16 ? kv_read_q4_tile_kernel<NG_, true> : kv_read_q4_tile_kernel<NG_, false>; \
      return launch_behind("kv_read_q4", kernel, grid, kQ4RowWarps * 32, 0, st, c.pool, c.slots, c.k, c.v, c.rows, hkv, tiles, \
                           c.num_slots, per); \
    }
    ICB_Q4_SIZES(ICB_RUN)
#undef ICB_RUN
  } else {
    const long long total = c.rows * hkv * (hd / 4), blocks = (total + 255) / 256;
    if (blocks > 0x7fffffffLL) return -3;
    auto kernel = c.dtype == kBF16 ? kv_read_q4_kernel<true> : kv_read_q4_kernel<false>;
    return launch_behind("kv_read_q4", kernel, (unsigned)blocks, 256, 0, st, c.pool, c.slots, c.k, c.v, total, hkv, hd, tiles,
                         c.num_slots);
  }
}
