// Rows of the 4-bit paged key / value cache (format: q4.cuh): quantise and write, read back.
//
// Quantisation of a group of 32 elements: scale = m / -8 rounded to fp16, m the element of largest magnitude (the largest
// if the smallest is as far from zero), so that m itself is code 0 and the other end of the range reaches code 15;
// n = clamp(round(x / scale), -8, 7) + 8, ties to even. x has at most 11 significant bits and scale at most 11, so a
// quotient that is not a tie differs from it by at least 2^-15 of its value: rounding the correctly rounded fp32 quotient
// gives the same code as exact arithmetic. The quotient is formed from the correctly rounded reciprocal with one residual
// correction (Markstein's theorem), which is exact in that sense and costs two multiply-adds.
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

__device__ __forceinline__ uint32_t q4_code(float x, float scale, float inv) {
  const float y0 = x * inv;
  const float y = fabsf(y0) < 64.f ? fmaf(fmaf(-y0, scale, x), inv, y0) : y0;
  return (uint32_t)(min(max(__float2int_rn(y), -8), 7) + 8);   // NaN converts to 0: code 8
}

// A thread takes 8 neighbouring elements of a token's keys (chunks 0 .. hd / 8 - 1) or values (the rest); the four threads
// of a group are neighbours.
template <bool BF16>
__global__ void __launch_bounds__(256)
kv_append_q4_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint8_t* __restrict__ pool,
                    const long long* __restrict__ slots, long long total, int hkv, int hd, int tiles, long long num_slots,
                    long long k_stride, long long v_stride) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per = hd / 8, ng = hd / 32;
  const int piece = (int)(i % (2 * per));
  const long long th = i / (2 * per);
  const int h = (int)(th % hkv);
  const long long t = th / hkv;
  const bool value = piece >= per;
  const int chunk = value ? piece - per : piece;
  long long slot = -1;
  if (i < total) slot = slots[t];
  const bool live = slot >= 0 && slot < num_slots;
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
  const __half sh = q4_scale(most, least);
  const float scale = __half2float(sh);
  const float inv = scale != 0.f ? __frcp_rn(scale) : 0.f;
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= q4_code(x[e], scale, inv) << (4 * e);
  uint8_t* tile = pool + q4_tile_of(slot, h, hkv, tiles, q4_tile_bytes(hd));
  const int tok = (int)(slot & 15);
  if (value) {
    uint8_t* half = tile + 8 * hd;
    *reinterpret_cast<uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk)) = (uint16_t)word;
    *reinterpret_cast<uint16_t*>(half + q4_value_at(ng, tok, 2 * chunk + 1)) = (uint16_t)(word >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(tile + q4_key_at(ng, tok, chunk)) = word;
  }
  if ((chunk & 3) == 0) {
    __half* scales = reinterpret_cast<__half*>(tile + 16 * hd) + tok * 2 * ng + (value ? ng : 0);
    scales[chunk >> 2] = sh;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256)
kv_read_q4_kernel(const uint8_t* __restrict__ pool, const long long* __restrict__ slots, uint16_t* __restrict__ k,
                  uint16_t* __restrict__ v, long long total, int hkv, int hd, int tiles, long long num_slots) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int per = hd / 8, ng = hd / 32;
  const int piece = (int)(i % (2 * per));
  const long long th = i / (2 * per);
  const int h = (int)(th % hkv);
  const long long t = th / hkv;
  const bool value = piece >= per;
  const int chunk = value ? piece - per : piece;
  const long long slot = slots[t];
  uint4 out = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0 && slot < num_slots) {
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
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = ((int)((word >> (8 * e)) & 15) - 8) * scale, hi = ((int)((word >> (8 * e + 4)) & 15) - 8) * scale;
      w[e] = BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
    }
    out = make_uint4(w[0], w[1], w[2], w[3]);
  }
  *reinterpret_cast<uint4*>((value ? v : k) + (t * hkv + h) * hd + chunk * 8) = out;
}

}  // namespace icb

using namespace icb;

// k, v: [T, hkv * hd] 16-bit rows of pitch k_stride / v_stride (16-byte aligned); pool: num_slots / (16 * tiles) pages of
// [hkv][tiles] tiles; a row whose slot is negative or outside the pool is left out. hd a multiple of 64.
ICB_API int icb_kv_append_q4(const void* k, const void* v, void* pool, const long long* slots, long long T, int hkv, int hd,
                             int tiles, long long num_slots, long long k_stride, long long v_stride, int dtype,
                             void* stream) {
  if (T <= 0) return 0;
  if (hkv < 1 || hd < 64 || hd % 64 || tiles < 1 || k_stride % 8 || v_stride % 8) return -2;
  const long long total = T * hkv * (hd / 4), blocks = (total + 255) / 256;
  if (blocks > 0x7fffffffLL) return -3;
  auto K = reinterpret_cast<const uint16_t*>(k), V = reinterpret_cast<const uint16_t*>(v);
  auto p = reinterpret_cast<uint8_t*>(pool);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == kBF16) kv_append_q4_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(K, V, p, slots, total, hkv, hd, tiles, num_slots, k_stride, v_stride);
  else if (dtype == kF16) kv_append_q4_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(K, V, p, slots, total, hkv, hd, tiles, num_slots, k_stride, v_stride);
  else return -4;
  return check_launch("kv_append_q4");
}

// The rows `slots` of the pool as 16-bit k, v [T, hkv * hd]; zeros for a slot outside the pool.
ICB_API int icb_kv_read_q4(const void* pool, const long long* slots, void* k, void* v, long long T, int hkv, int hd,
                           int tiles, long long num_slots, int dtype, void* stream) {
  if (T <= 0) return 0;
  if (hkv < 1 || hd < 64 || hd % 64 || tiles < 1) return -2;
  const long long total = T * hkv * (hd / 4), blocks = (total + 255) / 256;
  if (blocks > 0x7fffffffLL) return -3;
  auto K = reinterpret_cast<uint16_t*>(k), V = reinterpret_cast<uint16_t*>(v);
  auto p = reinterpret_cast<const uint8_t*>(pool);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == kBF16) kv_read_q4_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(p, slots, K, V, total, hkv, hd, tiles, num_slots);
  else if (dtype == kF16) kv_read_q4_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(p, slots, K, V, total, hkv, hd, tiles, num_slots);
  else return -4;
  return check_launch("kv_read_q4");
}
