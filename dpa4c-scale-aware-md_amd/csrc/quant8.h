// Loads, stores and roundings of the 8-bit forms (quant8.hip), for the kernels that read or write them.
#pragma once

#include "product.h"

namespace dpamd {

// t + kRound, |t| < 2^22, is t rounded to a whole number (ties to even), whose two's complement
// is in the sum's lowest bits.
constexpr float kRound = 12582912.0f;  // 1.5 * 2^23
__device__ __forceinline__ unsigned low_byte(float sum) { return __builtin_bit_cast(unsigned, sum) & 255u; }

// Eight elements from p on, the first `count` of them (at most eight, or none) there: zeros for the others.
template <int KIND>
__device__ __forceinline__ void load8(float (&v)[8], const typename ElemOf<KIND>::T* p, int count) {
  struct Eight {
    typename ElemOf<KIND>::T v[8];
  } s;
  if (count >= 8) {
    __builtin_memcpy(&s, p, sizeof(s));  // (the hardware takes addresses of any alignment)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32<KIND>(s.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? to_f32<KIND>(p[e]) : 0.0f;
  }
}
template <int KIND>
__device__ __forceinline__ void store8(typename ElemOf<KIND>::T* p, const float (&v)[8], int count) {
  struct Eight {
    typename ElemOf<KIND>::T v[8];
  } s;
  if (count >= 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s.v[e] = from_f32<KIND>(v[e]);
    __builtin_memcpy(p, &s, sizeof(s));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) p[e] = from_f32<KIND>(v[e]);
  }
}

// Eight kept columns from a multiple of eight on: q [rows][wide], then the fields [rows][wide / 32].
struct Kept8 {
  unsigned q[2];
  int field;
};
__device__ __forceinline__ Kept8 load_kept8(const unsigned char* kept, long rows, int wide, long row, int c0) {
  const unsigned long long q = *reinterpret_cast<const unsigned long long*>(kept + row * wide + c0);
  return Kept8{{(unsigned)q, (unsigned)(q >> 32)}, kept[rows * wide + row * (wide / 32) + c0 / 32]};
}
__device__ __forceinline__ float restore_one(int q, int field) {
  return field == 255 ? __builtin_bit_cast(float, 0x7fc00000u) : ldexpf((float)q, field - 133);
}
__device__ __forceinline__ void restore_kept8(const Kept8& k, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = restore_one((int)(signed char)(k.q[e / 4] >> (8 * (e % 4))), k.field);
}

}  // namespace dpamd
