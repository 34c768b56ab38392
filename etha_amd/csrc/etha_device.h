// Device helpers of the operators on local shards: element types, vectors at any byte address, conversions.
#ifndef ETHA_DEVICE_H
#define ETHA_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "etha_reshard.h"

namespace etha_device {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// The same vectors at any byte address: gfx950's global accesses need no alignment, so rows of odd widths take the
// same instructions as aligned ones.
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));

struct BF16 {
  typedef uint16_t bits;
  static __device__ float to_f32(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
  static __device__ uint16_t from_f32(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }  // nearest, ties to even
};
struct F16 {
  typedef uint16_t bits;
  static __device__ float to_f32(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
  static __device__ uint16_t from_f32(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};
struct F32 {
  typedef uint32_t bits;
  static __device__ float to_f32(uint32_t b) { return __builtin_bit_cast(float, b); }
  static __device__ uint32_t from_f32(float f) { return __builtin_bit_cast(uint32_t, f); }
};

// BYTES bytes at any address, BYTES a power of two up to 16; NT: not kept in the caches
template <int BYTES>
struct Raw;
template <> struct Raw<16> { typedef u32x4 type; typedef u32x4_any any; };
template <> struct Raw<8> { typedef u32x2 type; typedef u32x2_any any; };
template <> struct Raw<4> { typedef uint32_t type; typedef u32_any any; };
template <> struct Raw<2> { typedef uint16_t type; typedef u16_any any; };

template <int BYTES, bool NT = false>
__device__ inline typename Raw<BYTES>::type load_raw(const void* p) {
  typedef typename Raw<BYTES>::any any;
  if constexpr (NT) return __builtin_nontemporal_load((const any*)p);
  return *(const any*)p;
}
template <int BYTES, bool NT = false>
__device__ inline void store_raw(void* p, typename Raw<BYTES>::type v) {
  typedef typename Raw<BYTES>::any any;
  if constexpr (NT) __builtin_nontemporal_store(v, (any*)p);
  else *(any*)p = v;
}

// 16 bytes at p of which `left` exist; the others read as zero
template <int ES>
__device__ inline u32x4 load_part(const char* p, int64_t left) {
  if (left >= 16) return load_raw<16>(p);
  u32x4 v = {0, 0, 0, 0};
  if (left <= 0) return v;
  if constexpr (ES == 2) {
    #pragma unroll
    for (int i = 0; i < 8; i++)
      if (2 * i < left) v[i >> 1] |= (uint32_t)*(const uint16_t*)(p + 2 * i) << (16 * (i & 1));
  } else if constexpr (ES == 4) {
    #pragma unroll
    for (int i = 0; i < 4; i++)
      if (4 * i < left) v[i] = *(const uint32_t*)(p + 4 * i);
  } else {
    #pragma unroll
    for (int i = 0; i < 16; i++)
      if (i < left) v[i >> 2] |= (uint32_t)*(const uint8_t*)(p + i) << (8 * (i & 3));
  }
  return v;
}

// The elements of 16 bytes as fp32
template <typename T, int N>
__device__ inline void raw_to_f32(float (&out)[N], u32x4 raw) {
  static_assert(N * sizeof(typename T::bits) == 16, "one vector");
  typename T::bits e[N];
  __builtin_memcpy(e, &raw, 16);
  #pragma unroll
  for (int i = 0; i < N; i++) out[i] = T::to_f32(e[i]);
}

// N consecutive elements of type T as fp32; `n` of them exist (the rest read as zero)
template <typename T, int N, bool NT = false>
__device__ inline void load_f32(float (&out)[N], const typename T::bits* p, int64_t n) {
  typedef typename T::bits bits;
  constexpr int kBytes = N * (int)sizeof(bits), kPiece = kBytes > 16 ? 16 : kBytes, kPieces = kBytes / kPiece;
  constexpr int kPer = N / kPieces;
  if (n >= N) {
    #pragma unroll
    for (int i = 0; i < kPieces; i++) {
      const auto raw = load_raw<kPiece, NT>(p + i * kPer);
      bits e[kPer];
      __builtin_memcpy(e, &raw, kPiece);
      #pragma unroll
      for (int j = 0; j < kPer; j++) out[i * kPer + j] = T::to_f32(e[j]);
    }
  } else {
    #pragma unroll
    for (int j = 0; j < N; j++) out[j] = j < n ? T::to_f32(p[j]) : 0.f;
  }
}
template <typename T, int N, bool NT = false>
__device__ inline void store_f32(typename T::bits* p, const float (&v)[N], int64_t n) {
  typedef typename T::bits bits;
  constexpr int kBytes = N * (int)sizeof(bits), kPiece = kBytes > 16 ? 16 : kBytes, kPieces = kBytes / kPiece;
  constexpr int kPer = N / kPieces;
  if (n >= N) {
    #pragma unroll
    for (int i = 0; i < kPieces; i++) {
      bits e[kPer];
      #pragma unroll
      for (int j = 0; j < kPer; j++) e[j] = T::from_f32(v[i * kPer + j]);
      typename Raw<kPiece>::type raw;
      __builtin_memcpy(&raw, e, kPiece);
      store_raw<kPiece, NT>(p + i * kPer, raw);
    }
  } else {
    #pragma unroll
    for (int j = 0; j < N; j++)
      if (j < n) p[j] = T::from_f32(v[j]);
  }
}

// ---- rows to 8 bits ----------------------------------------------------------------------------------------------
// the largest magnitude so far by its bits: infinity is above all numbers, NaN above infinity
__device__ inline uint32_t largest_bits(const float (&v)[8], uint32_t top) {
  #pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t m = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    top = m > top ? m : top;
  }
  return top;
}
// the largest of each group of LANES lanes, in all of them
template <int LANES>
__device__ inline uint32_t group_max(uint32_t v) {
  #pragma unroll
  for (int d = LANES / 2; d; d >>= 1) {
    const uint32_t o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

// scale = max|x| * (1 / 127) in fp32; q = x / scale rounded half to even - of the exact quotient: with q0 next to it,
// r = x - q0 * scale is a multiple of ulp(scale) / 2 below scale and so an fp32 number, which the fused multiply-add
// gives exactly; comparing |r| with scale / 2 then settles the rounding.
struct RowScale {
  float scale, inverse;
  bool none, tiny;
  __device__ explicit RowScale(uint32_t top) {
    scale = __builtin_bit_cast(float, top) * (1.f / 127.f);
    none = !(scale > 0.f) || top >= 0x7f800000u;  // a row of zeros, or one that holds an infinity or NaN
    // a scale below the smallest normal number may have no finite inverse, and half of one below twice that may be no
    // number: the quotient is formed by division there
    tiny = scale < 2.4e-38f;
    inverse = 1.f / scale;
  }
  // x / scale rounded; near: x / scale, give or take a few roundings
  __device__ uint32_t value(float x, float near) const {
    float q = __builtin_rintf(near);
    const float r = __builtin_fmaf(-q, scale, x);
    const float twice = 2.f * __builtin_fabsf(r);
    // off by one, or a tie that went to the odd side
    if (twice > scale || (twice == scale && ((int)q & 1))) q += (r > 0.f) ? 1.f : -1.f;
    return (uint32_t)(int)__builtin_fmaxf(-127.f, __builtin_fminf(127.f, q)) & 255u;
  }
  // bytes 0 of eight words
  static __device__ u32x2 low_bytes(const float (&t)[8]) {
    u32x2 w;
    #pragma unroll
    for (int i = 0; i < 2; i++) {
      const auto bits = [&](int e) { return __builtin_bit_cast(uint32_t, t[4 * i + e]); };
      w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits(3), bits(2), 0x0c0c0400), __builtin_amdgcn_perm(bits(1), bits(0), 0x0c0c0400),
                                   0x05040100);
    }
    return w;
  }
  // Eight elements that came from type T.  Added to 1.5 * 2^23 a product is rounded to an integer, which the low byte of the
  // sum holds.  It is the wrong one only where what is left of x * inverse, which is off by at most 127 * 2^-24 < 2^-17, lies
  // within 2e-5 of one half: seldom in any of a wave's elements, but for bf16, whose few bits make such quotients common.
  // There, and otherwise, r says whether it is off by one; exact ties are left to the general way.  (56732 rows of 1024 in
  // fp16: 37 us, 40 us without the first way, 43 us the general way alone; 23040 rows of 2496 in bf16: 48 us, 54 us alone.)
  template <typename T>
  __device__ u32x2 pack(const float (&v)[8]) const {
    u32x2 w = {0, 0};
    if (none) return w;
    if (!tiny) {
      constexpr float kRound = 12582912.f;
      float t[8];
      if constexpr (!std::is_same_v<T, BF16>) {
        float left = 0.f;
        #pragma unroll
        for (int i = 0; i < 8; i++) {
          t[i] = __builtin_fmaf(v[i], inverse, kRound);
          left = __builtin_fmaxf(left, __builtin_fabsf(__builtin_fmaf(v[i], inverse, kRound - t[i])));
        }
        if (__ballot(left > 0.49998f) == 0) return low_bytes(t);
      }
      const float half = 0.5f * scale;
      bool tie = false;
      #pragma unroll
      for (int i = 0; i < 8; i++) {
        const float sum = __builtin_fmaf(v[i], inverse, kRound);
        const float r = __builtin_fmaf(kRound - sum, scale, v[i]);
        t[i] = sum + (__builtin_fabsf(r) > half ? __builtin_copysignf(1.f, r) : 0.f);
        tie |= __builtin_fabsf(r) == half;
      }
      if (__ballot(tie) == 0) return low_bytes(t);
    }
    #pragma unroll
    for (int i = 0; i < 8; i++) w[i >> 2] |= value(v[i], tiny ? v[i] / scale : v[i] * inverse) << (8 * (i & 3));
    return w;
  }
};

}  // namespace etha_device

// ---- host ----
// Calls f with the tag of the element type (checked before).
template <typename F>
inline void with_type(uint32_t dtype, F&& f) {
  if (dtype == ETHA_F32) f(etha_device::F32{});
  else if (dtype == ETHA_BF16) f(etha_device::BF16{});
  else f(etha_device::F16{});
}

#endif  // ETHA_DEVICE_H
