// Tile products on the matrix cores: C[m][n] = sum_k A(m, k) B(n, k), with an
// epilogue on the sums. The products of the gated block (gated.hip), for bf16, f16 and
// fp32 operands (v_mfma_f32_16x16x32_bf16 / _f16, v_mfma_f32_16x16x4_f32), and those of 8-bit integers
// (product8.hip, v_mfma_i32_16x16x64_i8).
#pragma once

#include <type_traits>

#include "common.h"
#include "ops.h"

namespace dpamd {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));

enum ElemKind { kBf16 = 0, kF16 = 1, kF32 = 2, kI8 = 3 };
template <int KIND>
struct ElemOf {
  using T = unsigned short;
};
template <>
struct ElemOf<kF32> {
  using T = float;
};
template <>
struct ElemOf<kI8> {
  using T = signed char;
};

// v rounded to the kind's 16 bits (to nearest, ties to even)
template <int KIND>
__device__ __forceinline__ unsigned short to16(float v) {
  if constexpr (KIND == kF16)
    return __builtin_bit_cast(unsigned short, (_Float16)v);
  else
    return __builtin_bit_cast(unsigned short, (__bf16)v);
}
template <int KIND>
__device__ __forceinline__ float to_f32(typename ElemOf<KIND>::T v) {
  if constexpr (KIND == kF32)
    return v;
  else if constexpr (KIND == kF16)
    return (float)__builtin_bit_cast(_Float16, v);
  else
    return __builtin_bit_cast(float, (unsigned)v << 16);
}
template <int KIND>
__device__ __forceinline__ typename ElemOf<KIND>::T from_f32(float v) {
  if constexpr (KIND == kF32)
    return v;
  else
    return to16<KIND>(v);
}

// v + that of another lane, in one instruction (DPP): within quads, halves of rows and rows of 16 lanes
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// The sum over a row of 16 lanes, in each of them.
__device__ __forceinline__ float sum_rows16(float v) {
  return add_dpp<0x140>(add_dpp<0x141>(add_dpp<0x4E>(add_dpp<0xB1>(v))));
}

// Four consecutive elements, aligned to them.
template <int KIND>
__device__ __forceinline__ void put4(typename ElemOf<KIND>::T* p, const f4& v) {
  if constexpr (KIND == kF32) {
    *reinterpret_cast<f4*>(p) = v;
  } else {
    typedef unsigned short us4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<us4*>(p) = us4{to16<KIND>(v[0]), to16<KIND>(v[1]), to16<KIND>(v[2]), to16<KIND>(v[3])};
  }
}

// Four columns of one row of an output, `count` of them inside it; FULL: all four, and aligned.
template <int KIND, bool FULL>
__device__ __forceinline__ void put_row4(void* out, long at, const f4& v, int count) {
  auto* o = static_cast<typename ElemOf<KIND>::T*>(out) + at;
  if constexpr (FULL) {
    put4<KIND>(o, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) o[e] = from_f32<KIND>(v[e]);
  }
}

// The activation a(g) and its derivative: tanh, silu g s(g), gelu g Phi(g), on the hardware's
// base-2 exponential and reciprocal (about 1 ulp each). tanh from q = 2 / (exp(2 |g|) + 1): 1 - q, which
// cancels where g is small, and there (below 0.625) an odd polynomial, fitted to 4e-9 of tanh;
// the derivative 1 - tanh^2 = q (2 - q) at any g. Relative errors in 32 bits: tanh 1.8e-7, the derivative
// 6e-7 up to |g| = 3 and 1e-6 at 9 (the exponent's rounding). silu to about 2e-7 of max(1, |g|). Phi
// below 1.25 as 1/2 + g R(g^2), beyond from Phi(-|g|) = exp(-g^2 / 2) (b1 t + .. + b7 t^7),
// t = 1 / (1 + 0.4 |g| / sqrt 2), which shares its exponential with the derivative; R and the b are fitted
// to 1e-8 and 4e-8 of Phi(-|g|) (least squares reweighted to an even error). gelu is off by 1.5e-7 of itself
// below 0.625, 7e-7 up to 3 and 4e-6 at -9 (the exponent's rounding). With the library's expf, tanhf,
// erff and a division the epilogues below issued about four times the instructions.
template <int ACT>
__device__ __forceinline__ void activate(float g, float& a, float& da) {
  constexpr float kLog2e = 1.4426950408889634f;
  if constexpr (ACT == kActTanh) {
    const float z = fabsf(g), s = g * g;
    const float e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * z);
    const float q = 2.0f * e * __builtin_amdgcn_rcpf(1.0f + e);
    const float odd =
        -0.33333282f + s * (0.13331442f + s * (-0.05373971f + s * (0.02063909f + s * -0.00570499f)));
    a = z < 0.625f ? g + g * s * odd : copysignf(1.0f - q, g);
    da = q * (2.0f - q);
  } else if constexpr (ACT == kActSilu) {
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
    a = g * p;
    da = p * (1.0f + g * (1.0f - p));
  } else {
    const float s = g * g;
    const float e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * s);
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.28284271f * fabsf(g));
    const float tail =
        0.112813413f +
        t * (0.113347933f +
             t * (0.0993796512f +
                  t * (0.106567279f + t * (0.00404826971f + t * (0.121886708f + t * -0.0581642948f)))));
    const float q = t * tail * e;  // Phi(-|g|)
    const float r =
        0.398942239f +
        s * (-0.0664897763f +
             s * (0.00997082248f + s * (-0.00118178294f + s * (0.000109763437f + s * -6.51857155e-06f))));
    const float p = fabsf(g) < 1.25f ? 0.5f + g * r : g < 0.0f ? q : 1.0f - q;
    a = g * p;
    da = p + g * e * 0.39894228040143268f;
  }
}
__device__ __forceinline__ void activate4(int act, const f4& g, f4& a, f4& da) {
  auto all = [&](auto k) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x, y;
      activate<decltype(k)::value>(g[r], x, y);
      a[r] = x;
      da[r] = y;
    }
  };
  if (act == kActTanh)
    all(std::integral_constant<int, kActTanh>{});
  else if (act == kActSilu)
    all(std::integral_constant<int, kActSilu>{});
  else
    all(std::integral_constant<int, kActGelu>{});
}

// The same for results of 16 bits that are formed element by element (the norm, the 8-bit products), whose
// vector instructions bound them: gelu's Phi(-|g|) as above at any g, by six terms in t = 1 / (1 + 0.3 |g|), fitted to
// 2.2e-7 and, where it is small, to 2.2e-5 of itself (half a step of f16 is 2.4e-4), so that gelu keeps its
// digits where it vanishes. gelu is off by 2.2e-7 of max(1, |g|), its derivative by 2.2e-7: 22 instructions for 30
// (forward; a rate of 4 counted as 4).
template <int KIND, int ACT>
__device__ __forceinline__ void activate_as(float g, float& a, float& da) {
  if constexpr (KIND == kF32 || ACT != kActGelu) {
    activate<ACT>(g, a, da);
  } else {
    const float e = __builtin_amdgcn_exp2f(-0.72134752f * (g * g));
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.3f * fabsf(g));
    const float tail =
        0.12006781f +
        t * (0.113619839f + t * (0.145477321f + t * (-0.0207191556f + t * (0.220416122f + t * -0.0788621576f))));
    const float q = t * tail * e;
    const float p = g < 0.0f ? q : 1.0f - q;
    a = g * p;
    da = p + g * e * 0.39894228040143268f;
  }
}

// ---- epilogues on four consecutive columns of one row, shared by the products and
// by the sums over slices of K --------------------------------------------------------

// The four columns are `count` of the output's (and the rest beyond it); FULL: all four, and
// aligned.

// h = a(g) u (zeros beyond the output)
template <bool FULL>
__device__ __forceinline__ f4 gate_value(int act, int count, const f4& g, const f4& u) {
  f4 a, da, v;
  activate4(act, g, a, da);
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = FULL || r < count ? a[r] * u[r] : 0.0f;
  return v;
}

// g and u of four columns are kept for the backward in 32 bits, so that what it forms from
// them is rounded once: all of g, and all of u `plane` floats on. (As pairs the lanes' 16 bytes of
// one instruction lay 32 apart.)
struct Kept {
  f4 g, u;
};
template <bool FULL>
__device__ __forceinline__ void put_kept(float* kept, long plane, int count, const f4& g, const f4& u) {
  if constexpr (FULL) {
    // (the hardware takes unaligned addresses)
    __builtin_memcpy(kept, &g, sizeof(g));
    __builtin_memcpy(kept + plane, &u, sizeof(u));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < count) {
        kept[r] = g[r];
        kept[plane + r] = u[r];
      }
  }
}
// as the forward kept them (zeros beyond the output)
template <bool FULL>
__device__ __forceinline__ Kept load_kept(const float* kept, long plane, int count) {
  Kept k;
  if constexpr (FULL) {
    __builtin_memcpy(&k.g, kept, sizeof(k.g));
    __builtin_memcpy(&k.u, kept + plane, sizeof(k.u));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      k.g[r] = r < count ? kept[r] : 0.0f;
      k.u[r] = r < count ? kept[plane + r] : 0.0f;
    }
  }
  return k;
}

// From dh and the kept g, u: dg = dh u a'(g), du = dh a(g) and h again.
struct GateGrad {
  f4 h, dg, du;
};
template <bool FULL>
__device__ __forceinline__ GateGrad gate_grad(int act, int count, const f4& dh, const Kept& k) {
  GateGrad o;
  f4 a, da;
  activate4(act, k.g, a, da);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const bool in = FULL || r < count;
    o.h[r] = in ? a[r] * k.u[r] : 0.0f;
    o.du[r] = in ? dh[r] * a[r] : 0.0f;
    o.dg[r] = in ? dh[r] * k.u[r] * da[r] : 0.0f;
  }
  return o;
}
template <int KIND>
__device__ __forceinline__ void put_gate_grad(const EpiArgs& e, long at, const GateGrad& o) {
  using T = typename ElemOf<KIND>::T;
  if (e.h) put4<KIND>(static_cast<T*>(e.h) + at, o.h);
  put4<KIND>(static_cast<T*>(e.dg) + at, o.dg);
  put4<KIND>(static_cast<T*>(e.du) + at, o.du);
}

// Where a lane of group g (at column 4 g of a fragment of 16) puts the eight columns that put_pair
// gives it.
__device__ __forceinline__ int pair_at(int g) { return 16 * (g & 1) + 8 * (g >> 1) - 4 * g; }
// v and w are columns 4 g .. 4 g + 3 of two neighbouring fragments: rounded to 16 bits and traded
// between lane groups, so that each has eight consecutive columns, 8 (g >> 1) .. of fragment g & 1, and
// stores 16 bytes (whose rows are then whole 64-byte pieces: with 8 bytes a lane dx of 131,072 x 2048
// took 411 us, so 370).
template <int KIND>
__device__ __forceinline__ void put_pair(typename ElemOf<KIND>::T* p, const f4& v, const f4& w) {
  static_assert(KIND != kF32, "four of 32 bits are 16 bytes already");
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  unsigned out[4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned x = __builtin_bit_cast(unsigned, us2{to16<KIND>(v[2 * e]), to16<KIND>(v[2 * e + 1])});
    const unsigned y = __builtin_bit_cast(unsigned, us2{to16<KIND>(w[2 * e]), to16<KIND>(w[2 * e + 1])});
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, true, false);
    out[e] = r[0];
    out[2 + e] = r[1];
  }
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<u4*>(p) = u4{out[0], out[1], out[2], out[3]};
}

// ---- products of 8-bit integers -----------------------------------------------------------

// act(g), or g itself, for results of a kind
template <int KIND>
__device__ __forceinline__ f4 activated4(int act, const f4& g) {
  if (act == kActNone) return g;
  f4 v;
  auto all = [&](auto k) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float a, da;
      activate_as<KIND, decltype(k)::value>(g[r], a, da);
      v[r] = a;
    }
  };
  if (act == kActTanh)
    all(std::integral_constant<int, kActTanh>{});
  else if (act == kActSilu)
    all(std::integral_constant<int, kActSilu>{});
  else
    all(std::integral_constant<int, kActGelu>{});
  return v;
}
// A row's scale as two factors: with that of rows beyond 2^90 a sum (below 2^31) could leave fp32's range
// before the column's scale brings it back.
struct RowFactor {
  float first, last;
};
__device__ __forceinline__ RowFactor row_factor(float scale) {
  return scale >= 0x1p90f ? RowFactor{scale * 0x1p-32f, 0x1p32f} : RowFactor{scale, 1.0f};
}
// Four columns of a row from the integer sums: act(g), or act(g) u; each sum in fp32 times the row's scale
// and then the column's.
template <int KIND, bool GATE>
__device__ __forceinline__ f4 scaled4(int act, const f4& sums, const f4& other, const RowFactor& row, const f4& col,
                                      const f4& col_other) {
  const i4 s = __builtin_bit_cast(i4, sums), o = __builtin_bit_cast(i4, other);
  f4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)s[e] * row.first * col[e] * row.last;
  v = activated4<KIND>(act, v);
  if constexpr (GATE) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= (float)o[e] * row.first * col_other[e] * row.last;
  }
  return v;
}
// Four consecutive elements at any alignment (which the hardware takes).
template <int KIND>
__device__ __forceinline__ void put_any4(typename ElemOf<KIND>::T* p, const f4& v) {
  struct Four {
    typename ElemOf<KIND>::T v[4];
  } s;
#pragma unroll
  for (int e = 0; e < 4; ++e) s.v[e] = from_f32<KIND>(v[e]);
  __builtin_memcpy(p, &s, sizeof(s));
}
// Scales of four columns, `count` of them there.
__device__ __forceinline__ f4 scales4(const float* s, int count) {
  f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (count >= 4) {
    __builtin_memcpy(&v, s, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < count) v[e] = s[e];
  }
  return v;
}
// A wave's sums: rows m0 + 16 i, columns n0 + 16 j .. + 3 of its lanes; acc[i][NG + j] the second matrix's.
template <int MI, int NG, bool GATE, int NJ>
__device__ __forceinline__ void scaled_out(const ProductArgs& p, const f4 (&acc)[MI][NJ], int m0, int n0, int g,
                                           bool inside) {
  f4 col[NG], other[NG];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    col[j] = scales4(p.col_scale[0] + n0 + j * 16, p.N - n0 - j * 16);
    other[j] = GATE ? scales4(p.col_scale[1] + n0 + j * 16, p.N - n0 - j * 16) : f4{};
  }
  float scale[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) scale[i] = p.row_scale[min(m0 + i * 16, p.M - 1)];
  auto emit = [&](auto kind) {
    constexpr int OUT = decltype(kind)::value;
    auto value = [&](int i, int j) {
      return scaled4<OUT, GATE>(p.act, acc[i][j], acc[i][GATE ? NG + j : j], row_factor(scale[i]), col[j], other[j]);
    };
    using T = typename ElemOf<OUT>::T;
    const long step = 16 * p.ldo[0];
    long at = m0 * p.ldo[0] + n0;
    if constexpr (OUT != kF32 && NG % 2 == 0) {
      if (inside && p.wide[0]) {
        at += pair_at(g);
#pragma unroll
        for (int i = 0; i < MI; ++i, at += step)
#pragma unroll
          for (int j = 0; j < NG; j += 2)
            put_pair<OUT>(static_cast<T*>(p.out[0]) + at + j * 16, value(i, j), value(i, j + 1));
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < MI; ++i, at += step)
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const f4 v = value(i, j);
        if (inside || (m0 + i * 16 < p.M && n0 + j * 16 + 4 <= p.N))
          put_any4<OUT>(static_cast<T*>(p.out[0]) + at + j * 16, v);
        else if (m0 + i * 16 < p.M && n0 + j * 16 < p.N)
          put_row4<OUT, false>(p.out[0], at + j * 16, v, p.N - n0 - j * 16);
      }
  };
  if (p.out_elem == kF32)
    emit(std::integral_constant<int, kF32>{});
  else if (p.out_elem == kF16)
    emit(std::integral_constant<int, kF16>{});
  else
    emit(std::integral_constant<int, kBf16>{});
}

// ---- the product ------------------------------------------------------------------------

// Operand layouts: rows with k contiguous (kRowK), or k rows with the operand's rows
// contiguous (kColK: element (r, k) at k ld + r).
enum Layout { kRowK = 0, kColK = 1 };

typedef __attribute__((address_space(3))) s4v lds_s4;

// 16 bytes a lane from base + offset straight into LDS: lane l's to the LDS address lds + 16 l
// (base and lds are wave-uniform; tile_landed() is the wait). Written as an instruction,
// which has no register result, because the compiler waits for every such load that it
// knows of before any transposing LDS read, as it can not tell that they are of different tiles:
// with the builtin each row of k-strided fragments waited for the loads issued just before it.
// (m0 is a register that a statement may not name as changed; nothing else in these kernels uses it.
// The s_nop is the wait state between m0's move and the load. The compiler inserts none for what a
// statement reads: had a vector instruction written the address, the load would need five after it. In
// all kernels built the address comes from scalar instructions, which need none, and
// tests/test_ops_listing.py holds the build to it; five states in the statement cost 1 % of the large products.)
__device__ __forceinline__ void load_to_lds(const char* base, unsigned offset, unsigned lds) {
  // (both in scalar registers, whatever the compiler knows of them)
  lds = __builtin_amdgcn_readfirstlane(lds);
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)(size_t)base);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((size_t)base >> 32));
  const size_t at = ((size_t)hi << 32) | lo;
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(offset), "s"(at), "s"(lds)
      : "memory");
}
// Every load_to_lds of this wave has landed, and after the barrier every wave's; all
// LDS reads before it are done.
__device__ __forceinline__ void tile_landed() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// One operand's tile in LDS: ROWS rows by 128 bytes of k (BK = 64 or 32 elements of EB bytes), in
// SUB side-by-side parts of ROWS / SUB rows that come from as many matrices.
//
// kRowK: rows of 128 bytes, whose 16-byte chunks are permuted by pairs, so that the sixteen
// rows that a fragment read takes at one chunk lie in different banks (a read takes its lanes
// in the groups 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 of each half of the wave: eight rows
// at each of two neighbouring chunks).
// kColK: per part, BK rows of ROWS / SUB elements. 16 bits: read by the transposing LDS load, 32-byte
// units permuted by xor with (k & 3) + 4 ((k >> 3) & 3), so that the 4 k rows of each of the four lane
// groups of one read fall in different banks. 32 bits: read element by element, 64-byte
// units permuted by xor with (k >> 2) & 3 for the same.
// The tile is written by the direct global-to-LDS load, whose lanes fill 1 KB in lane
// order; the permutation is on the side of the global addresses.
template <int LAYOUT, int ROWS, int EB, int SUB, int WAVES>
struct TileOf {
  static constexpr int BK = 128 / EB, VE = 16 / EB;  // k of a tile, elements of a chunk
  static constexpr int kBytes = ROWS * 128;
  static constexpr int kPart = ROWS / SUB;
  static constexpr int kLoads = kBytes / 1024 / WAVES;  // per wave
  static_assert(kLoads * 1024 * WAVES == kBytes, "a tile is whole 1 KB loads of every wave");
  static constexpr int kKRow = kPart * EB;               // bytes of one k row of a part (kColK)
  static constexpr int kUnits = kKRow / (EB == 2 ? 32 : 64);
  static constexpr int kPeriod = EB == 2 ? 32 : 16;      // k rows of one permutation

  static __device__ __forceinline__ int swz_row(int row) { return ((row / 2) & 3) << 1; }
  static __device__ __forceinline__ int swz_k(int k) {  // in chunks
    if constexpr (EB == 2)
      return (((k & 3) | (((k >> 3) & 3) << 2)) & (kUnits - 1)) << 1;
    else
      return (((k >> 2) & 3) & (kUnits - 1)) << 2;
  }
  // place of this lane in load q: part, row or k row, chunk
  static __device__ __forceinline__ void place(int q, int wave, int lane, int& part, int& row, int& chunk) {
    const int b = (q * WAVES + wave) * 1024 + lane * 16;
    if constexpr (LAYOUT == kRowK) {
      part = SUB == 1 ? 0 : b / 128 / kPart;
      row = SUB == 1 ? b / 128 : b / 128 % kPart;
      chunk = ((b / 16) % 8) ^ swz_row(row);
    } else {
      part = b / (kPart * 128);
      const int w = b % (kPart * 128);
      row = w / kKRow;
      chunk = ((w / 16) % (kKRow / 16)) ^ swz_k(row);
    }
  }
  // Byte offset of this lane's 16 bytes of load q from the part's origin at the step's k:
  // offset(kind(q)) + moved(q) rows of ld, the former in a register for each of kOffsets
  // kinds. (Rows, or k rows a period apart, differ by the uniform part alone.)
  static constexpr int kRows = LAYOUT == kRowK ? WAVES * 8 : WAVES * 1024 / kKRow;  // of one load of all waves
  static_assert(LAYOUT == kColK || (kRows % 8 == 0 && kPart % 8 == 0), "whole permutations a load");
  static_assert(LAYOUT == kColK || kPart % kRows == 0 || kRows == ROWS, "a load's rows lie alike in their parts");
  static constexpr int kOffsets =
      LAYOUT == kRowK || kRows >= kPeriod ? 1 : (kPeriod / kRows < kLoads ? kPeriod / kRows : kLoads);
  static constexpr __device__ int kind(int q) { return q % kOffsets; }
  // (Two spellings of the same rows, by what the compiler makes of them. 8-bit integers with the remainder and a 64-bit
  // difference in outside(): 16,384 x 8192 -> 2048 264 us, and 289 with the others' spelling. The others with neither: the
  // gate's gradient of 131,072 x 1600-240-240 152 us in 160 registers, and 166 in 172 with that of the integers.)
  static constexpr __device__ long moved(int q) {
    return LAYOUT == kRowK ? (SUB == 1 && EB != 1 ? q * kRows : (q * kRows) % kPart) : (q * kRows) % BK / kPeriod * kPeriod;
  }
  static __device__ __forceinline__ unsigned offset(int q, int wave, int lane, long ld, int rows_left) {
    int part, row, chunk;
    place(q, wave, lane, part, row, chunk);
    if constexpr (LAYOUT == kRowK) {
      return (unsigned)(row * ld * EB + chunk * 16);
    } else {
      const int left = (rows_left + VE - 1) / VE - 1;  // the last chunk of the row
      return (unsigned)(row * ld * EB + min(chunk, left) * 16);
    }
  }
  // whether the lane's 16 bytes of load q lie at or past the end of k
  static __device__ __forceinline__ bool past(int q, int wave, int lane, int k_left) {
    int part, row, chunk;
    place(q, wave, lane, part, row, chunk);
    return (LAYOUT == kRowK ? chunk * VE : row) >= k_left;
  }
  // or in a row past the operand's last (whose sums are not stored, whatever its tile row holds)
  static __device__ __forceinline__ bool outside(int q, int wave, int lane, int k_left, int rows_left) {
    int part, row, chunk;
    if constexpr (LAYOUT == kRowK) {
      place(0, wave, lane, part, row, chunk);
      using Rows = std::conditional_t<EB == 1, long, int>;
      return chunk * VE >= k_left || row >= rows_left - (Rows)moved(q);
    } else {
      place(q, wave, lane, part, row, chunk);
      return row >= k_left;
    }
  }
  // The fragment of rows r0 .. r0 + 15 (of part `part`) and half `kk` of the tile's k: lane
  // (g, c) holds row c. 16 bits: k 8 g .. 8 g + 7 of the 32. 32 bits: k 4 g .. 4 g + 3 of the
  // 16, of which element q is the operand of the q-th of four products.
  static __device__ __forceinline__ s8v frag(const char* tile, int part, int r0, int kk, int lane) {
    const int g = lane >> 4, c = lane & 15;
    if constexpr (LAYOUT == kRowK) {
      return *reinterpret_cast<const s8v*>(tile + (part * kPart + r0 + c) * 128 + (((kk * 4 + g) ^ swz_row(c)) * 16));
    } else if constexpr (EB == 2) {
      const int k = kk * 32 + 8 * g + (c >> 2);
      const int s = (((c >> 2) | (g << 2)) & (kUnits - 1)) ^ (r0 / 16);
      const char* p = tile + part * (kPart * 128) + k * kKRow + s * 32 + (c & 3) * 8;
      const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
      const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * kKRow));
      return s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      const char* p = tile + part * (kPart * 128) + (kk * 16 + 4 * g) * kKRow +
                      (((g & (kUnits - 1)) ^ (r0 / 16)) * 64) + c * 4;
      f4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const float*>(p + q * kKRow);
      return __builtin_bit_cast(s8v, v);
    }
  }
};

// acc[j] += the products of one row fragment and NJ column fragments (whose places are
// exchanged: a lane then holds four consecutive columns of one row). fp32: the four products
// of each j apart from each other, as one that waits for the last one's sum is issued late.
template <int KIND, int NJ>
__device__ __forceinline__ void multiply_row(f4 (&acc)[NJ], const s8v (&b)[NJ], s8v a) {
  if constexpr (KIND == kF32) {
    const f4 y = __builtin_bit_cast(f4, a);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] = mfma_f32(__builtin_bit_cast(f4, b[j])[q], y[q], acc[j]);
  } else if constexpr (KIND == kI8) {
    // (the sums are integers in the accumulators' bits)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      acc[j] = __builtin_bit_cast(
          f4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, b[j]), __builtin_bit_cast(i4, a),
                                                    __builtin_bit_cast(i4, acc[j]), 0, 0, 0));
  } else {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (KIND == kBf16)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, b[j]), __builtin_bit_cast(bf8, a),
                                                         acc[j], 0, 0, 0);
      else
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, b[j]), __builtin_bit_cast(h8, a),
                                                        acc[j], 0, 0, 0);
    }
  }
}

// Shape of a block's tile: BM rows by BN columns, WM by WN waves.
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
};

// EPI: kEpiStore, kEpiGate (two B matrices, BN / 2 columns of each), kEpiGateGrad, kEpiGateBack, kEpiGateOuts, kEpiGateOne (two); of 8-bit
// integers kEpiScale, kEpiScaleGate (two).
//
// A block takes tiles (and slices of K) one after another; the first two steps of the next one are
// loaded before the epilogue of the last, so that they arrive under it. Two stages of LDS.
//
// 16 bits, large products: bound by what the matrix cores reach while LDS is read beside them
// (0.6 of their cycles, 1090 to 1300 TFLOP/s; a large library product 1130 to 1600), and the
// epilogues with much to load and store by the bytes (one block a compute unit holds the large
// tiles, so that they do not run beside products). Steps on the way, training step of 8192 rows
// through 2048-8192-2048 in bf16 (kernels in turn): fragments read where they are used, operations of the
// library in the epilogues 4578 us; hardware exponentials, the kept g, u fetched a row ahead 3171;
// fragments read a half ahead, loads spread over the products 2676; one address and one test a
// row of the epilogue 2614; queued, 2373; 16 bytes a lane stored, g and u apart 2307; waves in
// their products at raised priority 2286. fp32: bound by
// the fp32 matrix cores (0.8 of their cycles). Few rows or columns: by a step's own chain of barrier,
// LDS reads and products, which slices of K and small tiles share out (four steps in LDS
// instead of two changed nothing).
template <int KIND, int LA, int LB, int EPI, class S>
__global__ __launch_bounds__(S::WM* S::WN * 64) void k_product(const ProductArgs p) {
  constexpr int SUB = EPI == kEpiGate || EPI == kEpiScaleGate || EPI == kEpiGateBack ||
                              EPI == kEpiGateOuts || EPI == kEpiGateOne
                          ? 2
                          : 1,
                EB = sizeof(typename ElemOf<KIND>::T), BK = 128 / EB;
  using T = typename ElemOf<KIND>::T;
  constexpr int WAVES = S::WM * S::WN, TM = S::BM / S::WM, TN = S::BN / S::WN;
  constexpr int MI = TM / 16, NJ = TN / 16;
  using TA = TileOf<LA, S::BM, EB, 1, WAVES>;
  using TB = TileOf<LB, S::BN, EB, SUB, WAVES>;
  constexpr int kStage = TA::kBytes + TB::kBytes;
  __shared__ __align__(1024) char lds[2 * kStage];
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)lds);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN, g = lane >> 4, c = lane & 15;
  const int K = p.K, per_seg = (K + BK - 1) / BK, steps = per_seg * p.segs;
  const long lda = EB * p.a[0].ld, ldb = EB * p.b[0].ld;  // bytes
  const long da = LA == kRowK ? 128 : BK * lda, db = LB == kRowK ? 128 : BK * ldb;

  // ---- a tile and its steps ----
  struct Item {
    int m0, n0, mat, slice, t0, t1;
  };
  // items in the order slice by slice, tiles in groups of eight row tiles by all column
  // tiles, so that the tiles under way on one XCD share rows and columns
  // (readfirstlane: quotients are formed on vector registers, and what is computed from them would be too)
  auto item_of = [&](int id) {
    Item it;
    const int tiles = p.tiles_m * p.tiles_n;
    it.slice = __builtin_amdgcn_readfirstlane(id / tiles);
    const int tile = id - it.slice * tiles, group = 8 * p.tiles_n;
    const int q = __builtin_amdgcn_readfirstlane(tile / group), in = tile - q * group;
    const int gm = min(8, p.tiles_m - 8 * q);
    const int tn = __builtin_amdgcn_readfirstlane(in / gm);
    it.mat = p.mats == 2 && tn >= p.tiles_n1;
    it.m0 = (8 * q + in - tn * gm) * S::BM;
    it.n0 = (tn - (it.mat ? p.tiles_n1 : 0)) * (S::BN / SUB);
    it.t0 = __builtin_amdgcn_readfirstlane((int)((long)steps * it.slice / p.split));
    it.t1 = __builtin_amdgcn_readfirstlane((int)((long)steps * (it.slice + 1) / p.split));
    return it;
  };
  const int items = p.tiles_m * p.tiles_n * p.split;
  int walk, walk_step = 1, walk_end = 0;
  if ((int)gridDim.x == items) {
    walk = __builtin_amdgcn_readfirstlane(xcd_swizzle().x);
  } else {
    const ChunkWalk w = xcd_chunks(items);
    walk = w.first, walk_step = w.step, walk_end = w.end;
  }
  if ((int)gridDim.x != items && walk >= walk_end) return;

  Item it = item_of(walk);
  unsigned oa[TA::kOffsets], ob[TB::kOffsets];
  const char *a0, *a1, *b0, *b1;
  auto aim = [&]() {
#pragma unroll
    for (int l = 0; l < TA::kOffsets; ++l) oa[l] = TA::offset(l, wave, lane, p.a[0].ld, p.M - it.m0);
#pragma unroll
    for (int l = 0; l < TB::kOffsets; ++l) ob[l] = TB::offset(l, wave, lane, p.b[0].ld, p.N - it.n0);
    const long ra = LA == kRowK ? it.m0 * lda : (long)EB * it.m0, rb = LB == kRowK ? it.n0 * ldb : (long)EB * it.n0;
    const bool pair = SUB == 2 || p.segs == 2;
    a0 = reinterpret_cast<const char*>(p.a[0].p) + ra;
    a1 = reinterpret_cast<const char*>(p.a[1].p) + ra;
    b0 = reinterpret_cast<const char*>(p.b[pair ? 0 : it.mat].p) + rb;
    b1 = reinterpret_cast<const char*>(p.b[pair ? 1 : it.mat].p) + rb;
  };

  // where a step's loads come from (wave-uniform); none of them past the slice's end
  // (the products then read on in a tile of which no one uses what they read)
  struct Cursor {
    const char *pa, *pb, *pb_second;
    int k_left;
  };
  auto cursor = [&](int t) {
    const bool seg = t >= per_seg;
    const int step = seg ? t - per_seg : t;
    return Cursor{(seg ? a1 : a0) + step * da, (SUB == 1 && seg ? b1 : b0) + step * db, b1 + step * db,
                  t < it.t1 ? K - step * BK : 0};
  };
  // One of a step's kLoads loads of this wave, by the lanes whose row and k are before the ends;
  // the 16 bytes past the end of k are zeroed by fill() (in the last step of a segment).
  constexpr int kLoads = TA::kLoads + TB::kLoads;
  auto slot = [&](int q) { return (q * WAVES + wave) * 1024; };
  auto issue = [&](int q, const Cursor& u, int to) {
    if (q < TA::kLoads) {
      if (TA::outside(q, wave, lane, u.k_left, p.M - it.m0)) return;
      load_to_lds(u.pa + TA::moved(q) * lda, oa[TA::kind(q)], lds0 + to + slot(q));
    } else {
      const int l = q - TA::kLoads;
      if (TB::outside(l, wave, lane, u.k_left, p.N - it.n0)) return;
      // (every lane of one load lies in one part: a part is whole loads)
      const bool part = SUB == 2 && slot(l) >= TB::kBytes / 2;
      load_to_lds((part ? u.pb_second : u.pb) + TB::moved(l) * ldb, ob[TB::kind(l)], lds0 + to + slot(q));
    }
  };
  auto fill = [&](const Cursor& u, int to) {
    if (u.k_left <= 0 || u.k_left >= BK) return;
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      if (q < TA::kLoads ? TA::past(q, wave, lane, u.k_left) : TB::past(q - TA::kLoads, wave, lane, u.k_left))
        *reinterpret_cast<f4*>(lds + to + slot(q) + lane * 16) = f4{0.0f, 0.0f, 0.0f, 0.0f};
  };
  auto load = [&](int t, int to) {
    const Cursor u = cursor(t);
#pragma unroll
    for (int q = 0; q < kLoads; ++q) issue(q, u, to);
    fill(u, to);
  };
  auto frag_a = [&](const char* tile, int i, int kk) { return TA::frag(tile, 0, wm * TM + i * 16, kk, lane); };
  auto frag_b = [&](const char* tile, int j, int kk) {
    return TB::frag(tile + TA::kBytes, SUB == 2 ? j / (NJ / 2) : 0,
                    SUB == 2 ? wn * (TN / 2) + (j % (NJ / 2)) * 16 : wn * TN + j * 16, kk, lane);
  };

  aim();
  load(it.t0, 0);
  load(it.t0 + 1, kStage);
  for (;;) {
    f4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    tile_landed();
    // Two halves of 64 bytes of k a step: a half's fragments are multiplied while the next half's
    // are read. A row's fragments are read again, for the next half, as soon as its products are
    // issued, and so have the other rows' products of time to arrive; the columns' fragments,
    // which every row needs, and the last rows', whose registers come free too late, have two sets of
    // registers. (Two sets of all spilled.) A step's loads go into the tile that all waves
    // have just read, once the step before it has landed: one barrier a step, in its middle.
    constexpr int LATE = MI >= 4 ? 2 : 0, EARLY = MI - LATE;
    s8v fa[EARLY], fl[2][LATE + 1], fb[2][NJ];
    auto half = [&](auto h_, const char* next, bool loads, const Cursor& u, int to) {
      constexpr int h = decltype(h_)::value, o = h ^ 1;
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[o][j] = frag_b(next, j, o);
      __builtin_amdgcn_sched_barrier(0);
      // (a wave in its products is served before one at its reads and barriers)
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        multiply_row<KIND, NJ>(acc[i], fb[h], i < EARLY ? fa[i < EARLY ? i : 0] : fl[h][i < EARLY ? 0 : i - EARLY]);
        if (i < EARLY) fa[i < EARLY ? i : 0] = frag_a(next, i, o);
        if (i < EARLY && i >= EARLY - LATE) fl[o][i - EARLY + LATE] = frag_a(next, i + LATE, o);
        if (loads) {
#pragma unroll
          for (int q = 0; q < kLoads; ++q)
            if (q * MI / kLoads == i) issue(q, u, to);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      // the reads have landed (a compiler-placed wait would come after the next reads and be for those too)
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb[0][j] = frag_b(lds, j, 0);
#pragma unroll
    for (int i = 0; i < MI; ++i)
      (i < EARLY ? fa[i < EARLY ? i : 0] : fl[0][i < EARLY ? 0 : i - EARLY]) = frag_a(lds, i, 0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    for (int t = it.t0; t < it.t1; ++t) {
      const int cur = ((t - it.t0) & 1) * kStage;
      const Cursor u = cursor(t + 2);
      half(std::integral_constant<int, 0>{}, lds + cur, false, u, cur);
      tile_landed();
      fill(u, cur);
      half(std::integral_constant<int, 1>{}, lds + (kStage - cur), true, u, cur);
    }

    // the next item's first loads, then this one's epilogue
    const Item done = it;
    walk += walk_step;
    const bool more = walk < walk_end;
    if (more) {
      it = item_of(walk);
      aim();
      __syncthreads();  // every wave has read its last
      load(it.t0, 0);
      load(it.t0 + 1, kStage);
    }
    // One test a wave for what lies inside the output, and one address a row where all does:
    // with tests, products of 64 bits and branches for every four columns the epilogue issued
    // several thousand instructions a wave, and took longer than eight steps of products.
    const int m0 = done.m0 + wm * TM + c, n0 = done.n0 + wn * (TN / SUB) + 4 * g;
    constexpr bool WIDE = KIND != kF32;  // pairs of fragments are stored together
    const bool inside = done.m0 + (wm + 1) * TM <= p.M && done.n0 + (wn + 1) * (TN / SUB) <= p.N;
    if (p.split > 1 || (EPI == kEpiStore && LB == kRowK && p.raw)) {
      // a slice's sums, columns in rows of ldp (a multiple of 4)
      const int sub = SUB == 2 ? 2 : p.mats;
      float* o = p.partial + (((long)done.slice * sub + done.mat) * p.M + m0) * p.ldp + n0;
      const long second = (long)p.M * p.ldp, row = 16 * p.ldp;
#pragma unroll
      for (int i = 0; i < MI; ++i, o += row)
#pragma unroll
        for (int j = 0; j < NJ / SUB; ++j)
          if (inside || (m0 + i * 16 < p.M && n0 + j * 16 < p.cols)) {
            *reinterpret_cast<f4*>(o + j * 16) = acc[i][j];
            if constexpr (SUB == 2) *reinterpret_cast<f4*>(o + second + j * 16) = acc[i][j + NJ / 2];
          }
    } else if constexpr (EPI == kEpiStore) {
      const long row = 16 * p.ldo[done.mat];
      long at = m0 * p.ldo[done.mat] + n0;
      void* out = p.out[done.mat];
      bool stored = false;
      if constexpr (WIDE && NJ % 2 == 0) {
        if (inside && p.wide[done.mat]) {
          stored = true;
          long w = at + pair_at(g);
#pragma unroll
          for (int i = 0; i < MI; ++i, w += row)
#pragma unroll
            for (int j = 0; j < NJ; j += 2)
              put_pair<KIND>(static_cast<T*>(out) + w + j * 16, acc[i][j], acc[i][j + 1]);
        }
      }
      if (stored) {
      } else if (inside && p.vec[done.mat]) {
#pragma unroll
        for (int i = 0; i < MI; ++i, at += row)
#pragma unroll
          for (int j = 0; j < NJ; ++j) put_row4<KIND, true>(out, at + j * 16, acc[i][j], 4);
      } else {
#pragma unroll
        for (int i = 0; i < MI; ++i, at += row)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            if (m0 + i * 16 < p.M && n0 + j * 16 < p.N)
              put_row4<KIND, false>(out, at + j * 16, acc[i][j], p.N - n0 - j * 16);
      }
    } else if constexpr (KIND == kI8) {
      scaled_out<MI, NJ / SUB, SUB == 2>(p, acc, m0, n0, g, inside);
    } else if constexpr (EPI == kEpiGate) {
      long h = m0 * p.epi.ldh + n0;
      float* kept = p.epi.saved ? p.epi.saved + ((long)m0 * p.N + n0) : nullptr;
      const long hrow = 16 * p.epi.ldh, krow = p.epi.saved ? 16l * p.N : 0, plane = (long)p.M * p.N;
      T* to = static_cast<T*>(p.epi.h);
      float* h32 = p.epi.h32;
      constexpr int NG = NJ / SUB;  // fragments of g, and as many of u
      if (inside) {
#pragma unroll
        for (int i = 0; i < MI; ++i, h += hrow, kept += krow) {
          f4 v[NG];
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            v[j] = gate_value<true>(p.act, 4, acc[i][j], acc[i][j + NG]);
            if (p.epi.saved) put_kept<true>(kept + j * 16, plane, 4, acc[i][j], acc[i][j + NG]);
          }
          if (h32) {
#pragma unroll
            for (int j = 0; j < NG; ++j) *reinterpret_cast<f4*>(h32 + h + j * 16) = v[j];
          } else if constexpr (WIDE && NG % 2 == 0) {
#pragma unroll
            for (int j = 0; j < NG; j += 2) put_pair<KIND>(to + h + pair_at(g) + j * 16, v[j], v[j + 1]);
          } else {
#pragma unroll
            for (int j = 0; j < NG; ++j) put4<KIND>(to + h + j * 16, v[j]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < MI; ++i, h += hrow, kept += krow)
#pragma unroll
          for (int j = 0; j < NG; ++j)
            if (m0 + i * 16 < p.M && n0 + j * 16 < p.cols) {
              const int count = p.N - n0 - j * 16;
              const f4 v = gate_value<false>(p.act, count, acc[i][j], acc[i][j + NG]);
              if (h32)
                *reinterpret_cast<f4*>(h32 + h + j * 16) = v;
              else
                put4<KIND>(to + h + j * 16, v);
              if (p.epi.saved) put_kept<false>(kept + j * 16, plane, count, acc[i][j], acc[i][j + NG]);
            }
      }
    } else if constexpr (EPI == kEpiGateBack) {
      // g and u are here, dh in memory: one number to read for each three to write, where the gate's
      // gradient after a gate that kept g and u for it moves 22 bytes for these 14 (bf16). The next sixteen
      // rows' dh are under way as the kept values are below.
      constexpr int NG = NJ / SUB;
      auto rows = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        const float* dh_at = p.epi.dh + ((long)m0 * p.epi.dh_ld + n0);
        long at = m0 * p.epi.ldh + n0;
        auto fetch = [&](int i, f4* d) {
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            d[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (FULL || (m0 + i * 16 < p.M && n0 + j * 16 < p.N)) {
              const float* s = dh_at + i * 16l * p.epi.dh_ld + j * 16;
              d[j] = *reinterpret_cast<const f4*>(s);
              for (int z = 1; z < p.epi.dh_slices; ++z) d[j] += *reinterpret_cast<const f4*>(s + z * p.epi.dh_plane);
            }
          }
        };
        f4 dh[2][NG];
        fetch(0, dh[0]);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          if (i + 1 < MI) fetch(i + 1, dh[(i + 1) & 1]);
          GateGrad o[NG];
#pragma unroll
          for (int j = 0; j < NG; ++j)
            o[j] = gate_grad<FULL>(p.act, p.N - n0 - j * 16, dh[i & 1][j], Kept{acc[i][j], acc[i][j + NG]});
          vmem_wait_all();
          const long row = at + i * 16 * p.epi.ldh;
          if constexpr (FULL && WIDE && NG % 2 == 0) {
            auto store = [&](void* out, auto member) {
#pragma unroll
              for (int j = 0; j < NG; j += 2)
                put_pair<KIND>(static_cast<T*>(out) + row + pair_at(g) + j * 16, o[j].*member, o[j + 1].*member);
            };
            if (p.epi.h) store(p.epi.h, &GateGrad::h);
            store(p.epi.dg, &GateGrad::dg);
            store(p.epi.du, &GateGrad::du);
          } else {
#pragma unroll
            for (int j = 0; j < NG; ++j)
              if (FULL || (m0 + i * 16 < p.M && n0 + j * 16 < p.cols)) put_gate_grad<KIND>(p.epi, row + j * 16, o[j]);
          }
        }
      };
      if (inside)
        rows(std::true_type{});
      else
        rows(std::false_type{});
    } else if constexpr (EPI == kEpiGateOuts || EPI == kEpiGateOne) {
      // dh from a few outputs' dy, here, and h dy summed over the wave's rows: neither g and u nor h meet
      // memory. (31,920 rows of 70-96-1 in fp32: 30 us with the join, against 38 for a gate that keeps g and u and the
      // kernels that read them.)
      constexpr int NG = NJ / SUB, O = EPI == kEpiGateOne ? 1 : kFewOutputs;
      const int outs = O == 1 ? 1 : p.epi.outs;
      float w[NG][4][O], sum[NG][4][O] = {};
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 0; k < O; ++k) {
            const int n = n0 + j * 16 + e;
            w[j][e][k] = k < outs && n < p.N
                             ? to_f32<KIND>(static_cast<const T*>(p.epi.wd)[n * p.epi.ld_down + k])
                             : 0.0f;
          }
      long at = m0 * p.epi.ldh + n0;
#pragma unroll
      for (int i = 0; i < MI; ++i, at += 16 * p.epi.ldh) {
        const int m = m0 + i * 16;
        const bool there = m < p.M;
        float dy[O];
#pragma unroll
        for (int k = 0; k < O; ++k)
          dy[k] = there && k < outs ? to_f32<KIND>(static_cast<const T*>(p.epi.dy)[m * p.epi.ld_dy + k]) : 0.0f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          f4 dh = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < O; ++k)
            if (k < outs)
#pragma unroll
              for (int e = 0; e < 4; ++e) dh[e] += dy[k] * w[j][e][k];
          const GateGrad o =
              gate_grad<false>(p.act, p.N - n0 - j * 16, dh, Kept{acc[i][j], acc[i][j + NG]});
          if (!there) continue;  // (rows past the last hold anything)
#pragma unroll
          for (int k = 0; k < O; ++k)
            if (k < outs)
#pragma unroll
              for (int e = 0; e < 4; ++e) sum[j][e][k] += o.h[e] * dy[k];
          if (n0 + j * 16 < p.cols) put_gate_grad<KIND>(p.epi, at + j * 16, o);
        }
      }
      if (p.epi.outs_partial) {
        float* out = p.epi.outs_partial + (long)(done.m0 / S::BM * S::WM + wm) * p.N * outs;
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < O; ++k)
              if (k < outs) {
                const float v = sum_rows16(sum[j][e][k]);
                const int n = n0 + j * 16 + e;
                if (c == 0 && n < p.N) out[(long)n * outs + k] = v;
              }
      }
    } else {
      // The kept g, u of the next sixteen rows are under way while these rows' values are
      // computed, and are waited for before the stores that follow them are issued (a wait
      // for a load issued before stores would be a wait for those too).
      auto rows = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        const float* kept_at = p.epi.saved + ((long)m0 * p.N + n0);
        const long plane = (long)p.M * p.N;
        long at = m0 * p.epi.ldh + n0;
        auto fetch = [&](int i, Kept* k) {
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            k[j] = FULL || (m0 + i * 16 < p.M && n0 + j * 16 < p.N)
                       ? load_kept<FULL>(kept_at + i * 16l * p.N + j * 16, plane, p.N - n0 - j * 16)
                       : Kept{};
        };
        Kept kept[2][NJ];
        fetch(0, kept[0]);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          if (i + 1 < MI) fetch(i + 1, kept[(i + 1) & 1]);
          GateGrad o[NJ];
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            o[j] = gate_grad<FULL>(p.act, p.N - n0 - j * 16, acc[i][j], kept[i & 1][j]);
          vmem_wait_all();
          const long row = at + i * 16 * p.epi.ldh;
          if constexpr (FULL && WIDE) {
            auto store = [&](void* out, auto member) {
#pragma unroll
              for (int j = 0; j < NJ; j += 2)
                put_pair<KIND>(static_cast<T*>(out) + row + pair_at(g) + j * 16, o[j].*member, o[j + 1].*member);
            };
            if (p.epi.h) store(p.epi.h, &GateGrad::h);
            store(p.epi.dg, &GateGrad::dg);
            store(p.epi.du, &GateGrad::du);
          } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
              if (FULL || (m0 + i * 16 < p.M && n0 + j * 16 < p.cols)) put_gate_grad<KIND>(p.epi, row + j * 16, o[j]);
          }
        }
      };
      if (inside)
        rows(std::true_type{});
      else
        rows(std::false_type{});
    }
    if (!more) return;
  }
}

// The slices' sums added up, and the epilogue: a block takes 256 / G quads of columns, G
// threads each, every thread a contiguous share of the slices in order, the shares
// joined in order through LDS. With one thread a quad the 249 slices of a 96 x 1 sum took
// 62 us, a chain of loads.
template <int KIND, int EPI>
__global__ __launch_bounds__(256) void k_join(const ProductArgs p) {
  constexpr bool PAIR = EPI == kEpiGate || EPI == kEpiGateBack;
  constexpr int SUB = PAIR ? 2 : 1;
  __shared__ f4 part[SUB][256];
  const int G = p.join, per = 256 / G;
  const int quads = p.ldp / 4, sub = PAIR ? 2 : p.mats;
  const long rows = PAIR ? p.M : (long)p.M * p.mats;
  const int slot = threadIdx.x % per, share = threadIdx.x / per;
  const long at = (long)blockIdx.x * per + slot;
  const bool in = at < rows * quads;
  const long row = in ? at / quads : 0;
  const int n = in ? (int)(at % quads) * 4 : 0;
  const long slice = (long)sub * p.M * p.ldp;
  const float* s = p.partial + row * p.ldp + n;
  const int z0 = p.split * share / G, z1 = p.split * (share + 1) / G;
  f4 v = {0, 0, 0, 0}, w = v;
  int z = z0;
  for (; z + 4 <= z1; z += 4) {
    f4 q[4], r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      q[k] = *reinterpret_cast<const f4*>(s + (z + k) * slice);
      if constexpr (SUB == 2) r[k] = *reinterpret_cast<const f4*>(s + (z + k) * slice + (long)p.M * p.ldp);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v += q[k];
      if constexpr (SUB == 2) w += r[k];
    }
  }
  for (; z < z1; ++z) {
    v += *reinterpret_cast<const f4*>(s + z * slice);
    if constexpr (SUB == 2) w += *reinterpret_cast<const f4*>(s + z * slice + (long)p.M * p.ldp);
  }
  if (G > 1) {
    part[0][threadIdx.x] = v;
    if constexpr (SUB == 2) part[SUB - 1][threadIdx.x] = w;
    __syncthreads();
    if (share) return;
    for (int k = 1; k < G; ++k) {
      v += part[0][k * per + slot];
      if constexpr (SUB == 2) w += part[SUB - 1][k * per + slot];
    }
  }
  if (!in) return;
  const int mat = PAIR ? 0 : (int)(row / p.M);
  const long m = PAIR ? row : row % p.M;
  const long plane = (long)p.M * p.N;
  if constexpr (EPI == kEpiGate) {
    const f4 h = gate_value<false>(p.act, p.N - n, v, w);
    if (p.epi.h32)
      *reinterpret_cast<f4*>(p.epi.h32 + m * p.epi.ldh + n) = h;
    else
      put4<KIND>(static_cast<typename ElemOf<KIND>::T*>(p.epi.h) + m * p.epi.ldh + n, h);
    if (p.epi.saved) put_kept<false>(p.epi.saved + (m * p.N + n), plane, p.N - n, v, w);
  } else if constexpr (EPI == kEpiGateBack) {
    f4 dh = {0, 0, 0, 0};
    if (n < p.N)
      for (int z = 0; z < p.epi.dh_slices; ++z)
        dh += *reinterpret_cast<const f4*>(p.epi.dh + z * p.epi.dh_plane + m * p.epi.dh_ld + n);
    put_gate_grad<KIND>(p.epi, m * p.epi.ldh + n, gate_grad<false>(p.act, p.N - n, dh, Kept{v, w}));
  } else if constexpr (EPI == kEpiGateGrad) {
    const Kept k = load_kept<false>(p.epi.saved + (m * p.N + n), plane, p.N - n);
    put_gate_grad<KIND>(p.epi, m * p.epi.ldh + n, gate_grad<false>(p.act, p.N - n, v, k));
  } else if (p.vec[mat] && n + 4 <= p.N)
    put_row4<KIND, true>(p.out[mat], m * p.ldo[mat] + n, v, 4);
  else
    put_row4<KIND, false>(p.out[mat], m * p.ldo[mat] + n, v, p.N - n);
}

}  // namespace dpamd
