// Device helpers of the operators on local shards: element types, vectors at any byte address, conversions.
#ifndef ETHA_DEVICE_H
#define ETHA_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>

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

}  // namespace etha_device

#endif  // ETHA_DEVICE_H
