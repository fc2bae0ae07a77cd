// Tile products on the 16-bit matrix cores: C[m][n] = sum_k A(m, k) B(n, k), with an
// epilogue on the fp32 sums. The products of the gated block (gated.hip), for 16-bit
// operands and for fp32 ones as three exact bf16 pieces (bf16x3.h).
#pragma once

#include "bf16x3.h"
#include "ops.h"

namespace dpamd {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));

// Element kinds: kBf16, kF16, and kF32 whose operands are three bf16 planes.
enum ElemKind { kBf16 = 0, kF16 = 1, kF32 = 2 };
template <int KIND>
constexpr int pieces() {
  return KIND == kF32 ? 3 : 1;
}

// v rounded to the kind's 16 bits (to nearest, ties to even)
template <int KIND>
__device__ __forceinline__ unsigned short to16(float v) {
  if constexpr (KIND == kF16)
    return __builtin_bit_cast(unsigned short, (_Float16)v);
  else
    return __builtin_bit_cast(unsigned short, (__bf16)v);
}

// One element of an operand: its 16 bits, or its three pieces a plane apart.
template <int KIND>
__device__ __forceinline__ void put_operand(unsigned short* p, long plane, float v) {
  if constexpr (KIND == kF32) {
    const __bf16 h = (__bf16)v;
    const float r1 = v - (float)h;
    const __bf16 m = (__bf16)r1;
    p[0] = __builtin_bit_cast(unsigned short, h);
    p[plane] = __builtin_bit_cast(unsigned short, m);
    p[2 * plane] = __builtin_bit_cast(unsigned short, (__bf16)(r1 - (float)m));
  } else {
    p[0] = to16<KIND>(v);
  }
}

// Four consecutive elements (p 8-byte aligned, plane a multiple of 4).
template <int KIND>
__device__ __forceinline__ void put_operand4(unsigned short* p, long plane, const float* v) {
  typedef unsigned short us4 __attribute__((ext_vector_type(4)));
  us4 q[3];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (KIND == kF32) {
      const __bf16 h = (__bf16)v[e];
      const float r1 = v[e] - (float)h;
      const __bf16 m = (__bf16)r1;
      q[0][e] = __builtin_bit_cast(unsigned short, h);
      q[1][e] = __builtin_bit_cast(unsigned short, m);
      q[2][e] = __builtin_bit_cast(unsigned short, (__bf16)(r1 - (float)m));
    } else {
      q[0][e] = to16<KIND>(v[e]);
    }
  }
#pragma unroll
  for (int s = 0; s < pieces<KIND>(); ++s) *reinterpret_cast<us4*>(p + s * plane) = q[s];
}

// Columns n .. n + 3 of one row of an output of the kind's own type. `vec`: the
// rows are aligned to four elements.
template <int KIND>
__device__ __forceinline__ void put_row4(void* out, long at, const float* v, int count, bool vec) {
  if constexpr (KIND == kF32) {
    float* o = static_cast<float*>(out) + at;
    if (vec && count >= 4) {
      *reinterpret_cast<f4*>(o) = f4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < count) o[e] = v[e];
    }
  } else {
    typedef unsigned short us4 __attribute__((ext_vector_type(4)));
    unsigned short* o = static_cast<unsigned short*>(out) + at;
    if (vec && count >= 4) {
      *reinterpret_cast<us4*>(o) = us4{to16<KIND>(v[0]), to16<KIND>(v[1]), to16<KIND>(v[2]), to16<KIND>(v[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < count) o[e] = to16<KIND>(v[e]);
    }
  }
}

// The activation a(g) and its derivative: tanh, silu g s(g), gelu g Phi(g).
__device__ __forceinline__ void activation(int act, float g, float& a, float& da) {
  if (act == kActTanh) {
    a = tanhf(g);
    da = 1.0f - a * a;
  } else if (act == kActSilu) {
    const float p = 1.0f / (1.0f + expf(-g));
    a = g * p;
    da = p * (1.0f + g * (1.0f - p));
  } else {
    const float p = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    a = g * p;
    da = p + g * expf(-0.5f * g * g) * 0.39894228040143268f;
  }
}

// ---- epilogues on four consecutive columns of one row, shared by the products and
// by the sums over slices of K --------------------------------------------------------

// h = a(g) u in operand form (columns N .. ldh - 1 are zeros), g and u kept for the
// backward in 32 bits, so that what it forms from them is rounded once.
template <int KIND>
__device__ __forceinline__ void epi_gate(const EpiArgs& e, int act, long m, int n, int N, const float* g,
                                         const float* u) {
  float h[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float a, da;
    activation(act, g[r], a, da);
    h[r] = n + r < N ? a * u[r] : 0.0f;
  }
  put_operand4<KIND>(e.h + m * e.ldh + n, e.plane_h, h);
  if (e.saved) {
    float* s = e.saved + 2 * (m * (long)N + n);
    if ((N & 1) == 0 && n + 4 <= N) {  // (n is a multiple of 4, N even: 16-byte aligned)
      *reinterpret_cast<f4*>(s) = f4{g[0], u[0], g[1], u[1]};
      *reinterpret_cast<f4*>(s + 4) = f4{g[2], u[2], g[3], u[3]};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < N) {
          s[2 * r] = g[r];
          s[2 * r + 1] = u[r];
        }
    }
  }
}

// From dh and the kept g, u: dg = dh u a'(g), du = dh a(g) and h again, in operand form.
template <int KIND>
__device__ __forceinline__ void epi_gate_grad(const EpiArgs& e, int act, long m, int n, int N, const float* dh) {
  const float* s = e.saved + 2 * (m * (long)N + n);
  float g[4], u[4];
  if ((N & 1) == 0 && n + 4 <= N) {
    const f4 p = *reinterpret_cast<const f4*>(s), q = *reinterpret_cast<const f4*>(s + 4);
    g[0] = p[0], u[0] = p[1], g[1] = p[2], u[1] = p[3];
    g[2] = q[0], u[2] = q[1], g[3] = q[2], u[3] = q[3];
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      g[r] = n + r < N ? s[2 * r] : 0.0f;
      u[r] = n + r < N ? s[2 * r + 1] : 0.0f;
    }
  }
  float h[4], dg[4], du[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float a, da;
    activation(act, g[r], a, da);
    const bool in = n + r < N;
    h[r] = in ? a * u[r] : 0.0f;
    du[r] = in ? dh[r] * a : 0.0f;
    dg[r] = in ? dh[r] * u[r] * da : 0.0f;
  }
  const long at = m * e.ldh + n;
  if (e.h) put_operand4<KIND>(e.h + at, e.plane_h, h);
  put_operand4<KIND>(e.dg + at, e.plane_h, dg);
  put_operand4<KIND>(e.du + at, e.plane_h, du);
}

// ---- the product ------------------------------------------------------------------------

// Operand layouts: rows with k contiguous (kRowK), or k rows with the operand's rows
// contiguous (kRowMajorK: element (r, k) at k ld + r).
enum Layout { kRowK = 0, kColK = 1 };

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;
typedef __attribute__((address_space(3))) s4v lds_s4;

__device__ const unsigned g_zero16[4] = {0, 0, 0, 0};

// One operand's tile in LDS: `ROWS` rows by BK of k, in SUB side-by-side parts of
// ROWS / SUB rows that come from as many matrices.
//
// kRowK: rows of BK elements; the row's 16-byte chunks are permuted by xor with
// the row's index among the rows that share the 64 banks' 256 bytes, so that the
// sixteen rows a fragment read takes at one chunk lie in different banks.
// kColK: per part, BK rows of ROWS / SUB elements, read by the transposing LDS load; 32-byte
// units permuted by xor with (k & 3) + 4 ((k >> 3) & 3): the 4 k rows of each of the four lane
// groups of one read fall in different banks.
// The tile is written by the direct global-to-LDS load, whose lanes fill 1 KB in lane
// order; the permutation is on the side of the global addresses.
template <int LAYOUT, int ROWS, int BK, int SUB, int WAVES>
struct TileOf {
  static constexpr int kBytes = ROWS * BK * 2;
  static constexpr int kPart = ROWS / SUB;
  static constexpr int kLoads = kBytes / 1024 / WAVES;  // per wave
  static_assert(kLoads * 1024 * WAVES == kBytes, "a tile is whole 1 KB loads of every wave");
  static constexpr int kChunks = BK / 8;
  static constexpr int kUnits = kPart / 16;

  static __device__ __forceinline__ int swz_row(int row) {
    return (row / (256 / (BK * 2))) & (kChunks - 1);
  }
  static __device__ __forceinline__ int swz_k(int k) {
    return ((k & 3) | (((k >> 3) & 3) << 2)) & (kUnits - 1);
  }
  // place of this lane in load q: part, row or k row, chunk of eight elements
  static __device__ __forceinline__ void place(int q, int wave, int lane, int& part, int& row, int& chunk) {
    const int b = (q * WAVES + wave) * 1024 + lane * 16;
    if constexpr (LAYOUT == kRowK) {
      row = b / (BK * 2);
      chunk = ((b / 16) % kChunks) ^ swz_row(row);
      part = row / kPart;
      row %= kPart;
    } else {
      constexpr int kPartBytes = kPart * BK * 2;
      part = b / kPartBytes;
      const int w = b % kPartBytes;
      row = w / (kPart * 2);
      chunk = ((w / 16) % (kPart / 8)) ^ (swz_k(row) << 1);
    }
  }
  // byte offset of this lane's 16 bytes of load q from the part's origin at the step's k
  static __device__ __forceinline__ unsigned offset(int q, int wave, int lane, long ld, int rows_left) {
    int part, row, chunk;
    place(q, wave, lane, part, row, chunk);
    if constexpr (LAYOUT == kRowK) {
      // rows past the end repeat the last one: their sums are not stored
      return (unsigned)(min(row, rows_left - 1) * ld * 2 + chunk * 16);
    } else {
      const int left = ((rows_left + 7) & ~7) - 8;
      return (unsigned)(row * ld * 2 + min(chunk * 8, left) * 2);
    }
  }
  // whether the lane's 16 bytes of load q lie at or past the end of k
  static __device__ __forceinline__ bool past(int q, int wave, int lane, int k_left) {
    int part, row, chunk;
    place(q, wave, lane, part, row, chunk);
    return (LAYOUT == kRowK ? chunk * 8 : row) >= k_left;
  }
  // the fragment of rows r0 .. r0 + 15 (of part `part`) and k kk * 32 .. + 31
  static __device__ __forceinline__ s8v frag(const char* tile, int part, int r0, int kk, int lane) {
    const int g = lane >> 4, c = lane & 15;
    if constexpr (LAYOUT == kRowK) {
      const int row = part * kPart + r0 + c;
      return *reinterpret_cast<const s8v*>(tile + row * (BK * 2) + (((kk * 4 + g) ^ swz_row(c)) * 16));
    } else {
      const int k = kk * 32 + 8 * g + (c >> 2);
      const int s = (((c >> 2) | (g << 2)) & (kUnits - 1)) ^ (r0 / 16);
      const char* p = tile + part * (kPart * BK * 2) + k * (kPart * 2) + s * 32 + (c & 3) * 8;
      const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
      const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * kPart * 2));
      return s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }
};

template <int KIND>
__device__ __forceinline__ f4 mfma16(s8v a, s8v b, f4 c) {
  if constexpr (KIND == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return mfma_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c);
}

// acc += the products of all pieces (the six down to 2^-18, smallest first)
template <int KIND>
__device__ __forceinline__ f4 mfma_all(const s8v* a, const s8v* b, f4 c) {
  if constexpr (KIND == kF32) {
    c = mfma16<KIND>(a[1], b[1], c);
    c = mfma16<KIND>(a[2], b[0], c);
    c = mfma16<KIND>(a[0], b[2], c);
    c = mfma16<KIND>(a[1], b[0], c);
    c = mfma16<KIND>(a[0], b[1], c);
  }
  return mfma16<KIND>(a[0], b[0], c);
}

// Shape of a block's tile: BM rows by BN columns by BK of k, WM by WN waves.
template <int BM_, int BN_, int BK_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_;
};

// EPI: kEpiStore, kEpiGate (two B matrices, BN / 2 columns of each), kEpiGateGrad.
// Two stages of LDS: the loads of step t + 1 are issued after the barrier that ends
// step t - 1 and land while step t's fragments are multiplied.
template <int KIND, int LA, int LB, int EPI, class S>
__global__ __launch_bounds__(S::WM* S::WN * 64) void k_product(const ProductArgs p) {
  constexpr int P = pieces<KIND>(), SUB = EPI == kEpiGate ? 2 : 1;
  constexpr int WAVES = S::WM * S::WN, TM = S::BM / S::WM, TN = S::BN / S::WN;
  constexpr int MI = TM / 16, NJ = TN / 16;
  using TA = TileOf<LA, S::BM, S::BK, 1, WAVES>;
  using TB = TileOf<LB, S::BN, S::BK, SUB, WAVES>;
  constexpr int kStage = P * (TA::kBytes + TB::kBytes);
  __shared__ __align__(1024) char lds[2 * kStage];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
  // blocks in groups of eight row tiles by all column tiles, consecutive ones on one XCD
  const int3 id = xcd_swizzle();
  const int group = 8 * p.tiles_n, q = id.x / group, in = id.x % group;
  const int gm = min(8, p.tiles_m - 8 * q);
  const int tm = 8 * q + in % gm, tn_all = in / gm;
  const int mat = tn_all / p.tiles_n1, tn = tn_all % p.tiles_n1;
  const int m0 = tm * S::BM, n0 = tn * (S::BN / SUB);
  const int per_seg = (p.K + S::BK - 1) / S::BK, steps = per_seg * p.segs;
  const int t0 = (int)((long)steps * id.y / p.split), t1 = (int)((long)steps * (id.y + 1) / p.split);

  unsigned oa[TA::kLoads], ob[TB::kLoads];
#pragma unroll
  for (int l = 0; l < TA::kLoads; ++l) oa[l] = TA::offset(l, wave, lane, p.a[0].ld, p.M - m0);
#pragma unroll
  for (int l = 0; l < TB::kLoads; ++l) ob[l] = TB::offset(l, wave, lane, p.b[mat].ld, p.N - n0);

  auto load = [&](int t, char* to) {
    const int seg = t >= per_seg, k0 = (t - seg * per_seg) * S::BK;
    const Operand& A = p.a[seg];
    const char* pa = reinterpret_cast<const char*>(A.p) +
                     2 * (LA == kRowK ? (long)m0 * A.ld + k0 : (long)k0 * A.ld + m0);
    const char* pb[SUB];
    long bplane = 0;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const Operand& B = p.b[SUB == 2 ? s : p.segs == 2 ? seg : mat];
      pb[s] = reinterpret_cast<const char*>(B.p) +
              2 * (LB == kRowK ? (long)n0 * B.ld + k0 : (long)k0 * B.ld + n0);
      bplane = B.plane;
    }
    const int k_left = p.K - k0;
    const bool tail = k_left < S::BK;
#pragma unroll
    for (int s = 0; s < P; ++s) {
#pragma unroll
      for (int l = 0; l < TA::kLoads; ++l) {
        const char* src = pa + 2 * s * A.plane + oa[l];
        if (tail && TA::past(l, wave, lane, k_left)) src = reinterpret_cast<const char*>(g_zero16);
        __builtin_amdgcn_global_load_lds((global_void*)src,
                                         (lds_void*)(to + s * TA::kBytes + (l * WAVES + wave) * 1024), 16, 0, 0);
      }
#pragma unroll
      for (int l = 0; l < TB::kLoads; ++l) {
        // (every lane of one load lies in one part: a part is whole loads)
        const int part = SUB == 1 ? 0 : (l * WAVES + wave) * 1024 / (TB::kBytes / SUB);
        const char* src = (part ? pb[SUB - 1] : pb[0]) + 2 * s * bplane + ob[l];
        if (tail && TB::past(l, wave, lane, k_left)) src = reinterpret_cast<const char*>(g_zero16);
        __builtin_amdgcn_global_load_lds(
            (global_void*)src, (lds_void*)(to + P * TA::kBytes + s * TB::kBytes + (l * WAVES + wave) * 1024), 16, 0, 0);
      }
    }
  };

  f4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};

  if (t0 < t1) load(t0, lds);
  for (int t = t0; t < t1; ++t) {
    char* cur = lds + ((t - t0) & 1) * kStage;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads of step t are in LDS
    __syncthreads();                     // and so are the other waves'; step t - 1 is read
    if (t + 1 < t1) load(t + 1, lds + ((t + 1 - t0) & 1) * kStage);
#pragma unroll
    for (int kk = 0; kk < S::BK / 32; ++kk) {
      s8v b[NJ][P];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int s = 0; s < P; ++s)
          b[j][s] = TB::frag(cur + P * TA::kBytes + s * TB::kBytes, SUB == 2 ? j / (NJ / 2) : 0,
                             SUB == 2 ? wn * (TN / 2) + (j % (NJ / 2)) * 16 : wn * TN + j * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        s8v a[P];
#pragma unroll
        for (int s = 0; s < P; ++s) a[s] = TA::frag(cur + s * TA::kBytes, 0, wm * TM + i * 16, kk, lane);
        // the operands change places: a lane then holds four consecutive columns of one row
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mfma_all<KIND>(b[j], a, acc[i][j]);
      }
    }
  }

  const int g = lane >> 4, c = lane & 15;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + wm * TM + i * 16 + c;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < NJ / SUB; ++j) {
      const int n = n0 + wn * (TN / SUB) + j * 16 + 4 * g;
      if (n >= p.cols) continue;
      float v[4], w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = acc[i][j][r];
        w[r] = acc[i][SUB == 2 ? j + NJ / 2 : j][r];
      }
      if (p.split > 1) {
        // a slice's sums, columns in rows of ldp (a multiple of 4)
        const int sub = SUB == 2 ? 2 : p.mats;
        float* o = p.partial + (((long)id.y * sub + mat) * p.M + m) * p.ldp + n;
        *reinterpret_cast<f4*>(o) = f4{v[0], v[1], v[2], v[3]};
        if constexpr (SUB == 2) *reinterpret_cast<f4*>(o + (long)p.M * p.ldp) = f4{w[0], w[1], w[2], w[3]};
      } else if constexpr (EPI == kEpiGate) {
        epi_gate<KIND>(p.epi, p.act, m, n, p.N, v, w);
      } else if constexpr (EPI == kEpiGateGrad) {
        epi_gate_grad<KIND>(p.epi, p.act, m, n, p.N, v);
      } else {
        put_row4<KIND>(p.out[mat], (long)m * p.ldo[mat] + n, v, p.N - n, p.vec[mat]);
      }
    }
  }
}

// The slices' sums added up in order, and the epilogue.
template <int KIND, int EPI>
__global__ __launch_bounds__(256) void k_join(const ProductArgs p) {
  const int quads = p.ldp / 4, sub = EPI == kEpiGate ? 2 : p.mats;
  const long rows = EPI == kEpiGate ? p.M : (long)p.M * p.mats;
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at >= rows * quads) return;
  const long row = at / quads;
  const int n = (int)(at % quads) * 4;
  const int mat = EPI == kEpiGate ? 0 : (int)(row / p.M);
  const long m = EPI == kEpiGate ? row : row % p.M;
  const long slice = (long)sub * p.M * p.ldp;
  const float* s = p.partial + row * p.ldp + n;
  f4 v = {0, 0, 0, 0}, w = v;
  for (int z = 0; z < p.split; ++z) {
    v += *reinterpret_cast<const f4*>(s + z * slice);
    if constexpr (EPI == kEpiGate) w += *reinterpret_cast<const f4*>(s + z * slice + (long)p.M * p.ldp);
  }
  float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {w[0], w[1], w[2], w[3]};
  if constexpr (EPI == kEpiGate)
    epi_gate<KIND>(p.epi, p.act, m, n, p.N, a, b);
  else if constexpr (EPI == kEpiGateGrad)
    epi_gate_grad<KIND>(p.epi, p.act, m, n, p.N, a);
  else
    put_row4<KIND>(p.out[mat], m * p.ldo[mat] + n, a, p.N - n, p.vec[mat]);
}

}  // namespace dpamd
