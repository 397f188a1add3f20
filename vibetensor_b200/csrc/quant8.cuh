// The 8-bit format shared by activation checkpoints and the key/value cache (sm_100a).
//
// A group of values x (128 neighbours of a row, or one head of one cached token) is held as
// eight-bit levels q and one float scale:
//
//   amax  = max |x|                        (a NaN counts as the largest magnitude)
//   scale = amax * fl(1 / top)             top = 127 (int8) or 448 (e4m3, its largest value)
//   q     = round(fl(x * fl(top / amax)))  to the nearest level, ties to even
//   x'    = q * scale
//
// One division per group and one multiply per value; every step is a correctly rounded fp32
// operation, so the levels are a function of the inputs alone.  |x * fl(top / amax)| is at most
// top * (1 + 2^-23), which rounds to top in both formats: no clamp.  A group whose amax is below
// 2^-119 is held as zeros (top / amax would overflow).  A group that holds a NaN or an infinity is
// held as zeros with a NaN for its scale: the whole group reads back as NaN.
//
// Rounding to int8 is an add of 1.5 * 2^23, whose sum's low byte is the level: the hardware's conversion
// runs at a quarter of an add's rate (silu_mul with both copies and its backward, [16384,8192] bf16:
// 2.4 % more with conversions).  Levels are widened by conversions; byte permutes and
// subtractions in their place made a cache read 27 % slower.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace vb {

constexpr int kQ8Group = VBT_B200_Q8_GROUP;  // values of a row that share a scale in a checkpoint

template <int F> __device__ __forceinline__ constexpr float q8_top() {
  return F == VBT_B200_Q8_INT8 ? 127.0f : 448.0f;
}

struct Q8Scale {
  float up;    // multiplies a value before rounding
  float down;  // multiplies a level when it is read back; what is stored
};
// amax_bits: the bit pattern of the largest magnitude (sign cleared), compared as an unsigned
// number so that infinities and NaN rank above every finite value
template <int F> __device__ __forceinline__ Q8Scale q8_scale(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  if (amax < 0x1p-119f) return {0.0f, 0.0f};
  if (amax_bits >= 0x7f800000u) return {0.0f, __uint_as_float(0x7fffffffu)};
  return {__fdiv_rn(q8_top<F>(), amax), __fmul_rn(amax, 1.0f / q8_top<F>())};
}
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// four values -> four bytes
template <int F> __device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d, float up) {
  a = __fmul_rn(a, up); b = __fmul_rn(b, up); c = __fmul_rn(c, up); d = __fmul_rn(d, up);
  uint32_t w;
  if constexpr (F == VBT_B200_Q8_INT8) {
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: the sum's last place is 1
    const uint32_t ia = __float_as_uint(__fadd_rn(a, kRound)), ib = __float_as_uint(__fadd_rn(b, kRound));
    const uint32_t ic = __float_as_uint(__fadd_rn(c, kRound)), id = __float_as_uint(__fadd_rn(d, kRound));
    w = __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    w = lo | (hi << 16);
  }
  return up == 0.0f ? 0u : w;  // a group with a NaN or an infinity
}
template <int F> __device__ __forceinline__ uint8_t q8_pack1(float a, float up) {
  return static_cast<uint8_t>(q8_pack4<F>(a, 0.f, 0.f, 0.f, up));
}
// four bytes -> four levels (not yet multiplied by the scale)
template <int F> __device__ __forceinline__ void q8_levels4(uint32_t w, float (&v)[4]) {
  if constexpr (F == VBT_B200_Q8_INT8) {
    const int32_t s = static_cast<int32_t>(w);
    v[0] = static_cast<float>(static_cast<int8_t>(s));
    v[1] = static_cast<float>(static_cast<int8_t>(s >> 8));
    v[2] = static_cast<float>(static_cast<int8_t>(s >> 16));
    v[3] = static_cast<float>(s >> 24);
  } else {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
}
template <int F> __device__ __forceinline__ float q8_level1(uint8_t b) {
  if constexpr (F == VBT_B200_Q8_INT8) return static_cast<float>(static_cast<int8_t>(b));
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// V bytes of levels as one load / store
template <int V> struct Q8Raw;
template <> struct Q8Raw<8> { using type = uint2; };
template <> struct Q8Raw<4> { using type = uint32_t; };
template <> struct Q8Raw<1> { using type = uint8_t; };

template <int F, int V> __device__ __forceinline__ void q8_store(uint8_t* dst, const float (&v)[V], float up) {
  static_assert(V == 8 || V == 4);
  if constexpr (V == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(q8_pack4<F>(v[0], v[1], v[2], v[3], up),
                                                q8_pack4<F>(v[4], v[5], v[6], v[7], up));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = q8_pack4<F>(v[0], v[1], v[2], v[3], up);
  }
}
// levels of V bytes held in a register, times the scale
template <int F, int V>
__device__ __forceinline__ void q8_widen(typename Q8Raw<V>::type raw, float scale, float (&v)[V]) {
  if constexpr (V >= 4) {
    uint32_t w[V / 4];
    if constexpr (V == 8) { w[0] = raw.x; w[1] = raw.y; } else { w[0] = raw; }
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      float l[4];
      q8_levels4<F>(w[q], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] = __fmul_rn(l[e], scale);
    }
  } else {
    v[0] = __fmul_rn(q8_level1<F>(raw), scale);
  }
}

// largest magnitude (as bits) over the LANES neighbouring lanes that hold one group
template <int LANES> __device__ __forceinline__ uint32_t lanes_max(uint32_t b) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, d));
  return b;
}
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
// The same from the stored values of a lane, W vectors of N.  16-bit types are compared two at a
// time in their own bit patterns, which are ordered like the values.
template <class T, int N, int W, int LANES>
__device__ __forceinline__ uint32_t group_mag(const Vec<T, N> (&v)[W]) {
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int e = 0; e < N; e += 2) m = max_halves(m, *reinterpret_cast<const uint32_t*>(&v[k].v[e]) & 0x7fff7fffu);
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) m = max_halves(m, __shfl_xor_sync(0xffffffffu, m, d));
    m = max(m & 0xffffu, m >> 16);
    const uint16_t h = static_cast<uint16_t>(m);
    return __float_as_uint(to_f(*reinterpret_cast<const T*>(&h)));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) m = max(m, mag_bits(to_f(v[k].v[e])));
    return lanes_max<LANES>(m);
  }
}

}  // namespace vb
