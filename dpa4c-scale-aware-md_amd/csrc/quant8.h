// Loads, stores and roundings of the 8-bit forms (quant8.hip), for the kernels that read or write them.
#pragma once

#include "product.h"

namespace dpamd {

// t + kRound, |t| < 2^22, is t rounded to a whole number (ties to even), whose two's complement
// is in the sum's lowest bits.
constexpr float kRound = 12582912.0f;  // 1.5 * 2^23
__device__ __forceinline__ unsigned low_byte(float sum) { return __builtin_bit_cast(unsigned, sum) & 255u; }

// s = max |x| / 127 and q = x (127 / max |x|) to nearest: both quotients are rounded to fp32, and the fused
// multiply-add rounds their product with x once, to a whole number (the sum's last digit is 1), so that q
// is the same on every machine. `top`: the bits of max |x|.
struct RowScale {
  float inv, scale;
};
__device__ __forceinline__ RowScale row_scale(unsigned top) {
  const float m = __builtin_bit_cast(float, top);
  if (top >= 0x7f800000u) return RowScale{0.0f, __builtin_bit_cast(float, 0x7fc00000u)};
  if (m < 0x1p-119f) return RowScale{0.0f, 0.0f};  // (below, the quotients leave fp32's range)
  return RowScale{127.0f / m, m / 127.0f};
}
__device__ __forceinline__ unsigned quant8(float x, float inv) {
  return low_byte(__builtin_fmaf(x, inv, kRound));
}
__device__ __forceinline__ unsigned long long quantize8(const float (&v)[8], float inv) {
  unsigned q[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e / 4] |= quant8(v[e], inv) << (8 * (e % 4));
  return q[0] | (unsigned long long)q[1] << 32;
}

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
// 16 bytes at the alignment of an element; with ONCE past the caches, for what is not read again soon
typedef unsigned u4any __attribute__((ext_vector_type(4), aligned(2)));
template <bool ONCE>
__device__ __forceinline__ void store16(void* p, const u4any& v) {
  if constexpr (ONCE)
    __builtin_nontemporal_store(v, static_cast<u4any*>(p));
  else
    *static_cast<u4any*>(p) = v;
}
template <int KIND, bool ONCE = false>
__device__ __forceinline__ void store8(typename ElemOf<KIND>::T* p, const float (&v)[8], int count) {
  struct Eight {
    typename ElemOf<KIND>::T v[8];
  } s;
  if (count >= 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s.v[e] = from_f32<KIND>(v[e]);
    struct Words {
      u4any w[sizeof(Eight) / 16];
    };
    const Words w = __builtin_bit_cast(Words, s);
#pragma unroll
    for (int k = 0; k < (int)(sizeof(Eight) / 16); ++k) store16<ONCE>(reinterpret_cast<char*>(p) + 16 * k, w.w[k]);
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
// 2^(field - 133): a subnormal number below field 7; NaN for 255
__device__ __forceinline__ float unit_of(int field) {
  return field == 255 ? __builtin_bit_cast(float, 0x7fc00000u) : ldexpf(1.0f, field - 133);
}
// (a product with a power of two is exact, down to fp32's smallest number, which the unit is a multiple of)
__device__ __forceinline__ void restore_kept8(const Kept8& k, float (&v)[8]) {
  const float unit = unit_of(k.field);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)(signed char)(k.q[e / 4] >> (8 * (e % 4))) * unit;
}

}  // namespace dpamd
