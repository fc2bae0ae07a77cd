// The gated block's down side for few outputs (an energy an atom, a vector): up to four
// columns fill a thirtieth of a tile, so these run on the vector units, where the bytes of
// h, and of the kept g and u, bound them.
//
//   k_outs_down: y = h w_down; a group of lanes a row of h, w_down in LDS. h comes in fp32 whatever the
//     type: it is rounded for the matrix cores alone.
//   k_outs_grad: from dy and the kept g, u a thread forms dh = dy w_down^T of four columns,
//     then dg, du and h, row after row of its block's slice, and keeps its sums of h dy in registers: h is
//     neither rounded nor stored.
//   k_outs_join: the slices' sums of d w_down added up, in order.
#include <algorithm>

#include "product.h"

namespace dpamd {

namespace {

// LANES: those that share a row
template <int KIND, int O, int LANES>
__global__ __launch_bounds__(256) void k_outs_down(const OutsArgs p) {
  using T = typename ElemOf<KIND>::T;
  constexpr int V = 4, U = 4;
  extern __shared__ __align__(16) float w[];  // [O][ldh], zeros beyond w_down
  const int ldh = (int)p.ldh;
#pragma unroll 4
  for (int c = threadIdx.x; c < ldh; c += 256)
#pragma unroll
    for (int k = 0; k < O; ++k)
      w[k * ldh + c] = c < p.f && k < p.o ? to_f32<KIND>(static_cast<const T*>(p.wd)[c * p.ld_down + k]) : 0.0f;
  __syncthreads();
  const int lane = threadIdx.x % LANES, chunks = ldh / V;
  for (long r0 = (long)blockIdx.x * (256 / LANES); r0 < p.rows; r0 += (long)gridDim.x * (256 / LANES)) {
    const long row = r0 + threadIdx.x / LANES;
    const float* h = p.h + std::min(row, p.rows - 1) * p.ldh;
    float acc[O] = {};
    auto add = [&](const f4& a, int q) {
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int k = 0; k < O; ++k) acc[k] += a[e] * w[k * ldh + q * V + e];
    };
    int q = lane;
    for (; q + (U - 1) * LANES < chunks; q += U * LANES) {
      f4 a[U];
#pragma unroll
      for (int u = 0; u < U; ++u) a[u] = *reinterpret_cast<const f4*>(h + (q + u * LANES) * V);
#pragma unroll
      for (int u = 0; u < U; ++u) add(a[u], q + u * LANES);
    }
    for (; q < chunks; q += LANES) add(*reinterpret_cast<const f4*>(h + q * V), q);
#pragma unroll
    for (int k = 0; k < O; ++k) {
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) acc[k] += __shfl_xor(acc[k], d, kWave);
      if (k == lane && k < p.o && row < p.rows)
        static_cast<T*>(p.y)[row * p.ld_y + k] = from_f32<KIND>(acc[k]);
    }
  }
}

// Blocks: slices of the rows by groups of p.quads quads of columns; 256 / p.quads rows at a time.
template <int KIND, int O>
__global__ __launch_bounds__(256) void k_outs_grad(const OutsArgs p) {
  using T = typename ElemOf<KIND>::T;
  __shared__ float part[256 * 4 * O];
  const int at_once = 256 / p.quads, slot = threadIdx.x / p.quads, quad = threadIdx.x % p.quads;
  const int c = (blockIdx.y * p.quads + quad) * 4, count = p.f - c;
  const long r0 = p.rows * blockIdx.x / gridDim.x, r1 = p.rows * (blockIdx.x + 1) / gridDim.x;
  const long plane = p.rows * p.f;
  float w[4][O], acc[4][O] = {};
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int k = 0; k < O; ++k)
      w[e][k] = e < count && k < p.o ? to_f32<KIND>(static_cast<const T*>(p.wd)[(c + e) * p.ld_down + k]) : 0.0f;
  if (slot < at_once && c < p.ldh) {
    struct Row {
      Kept kept;
      float dy[O];
    };
    auto fetch = [&](long r) {
      Row x;
      const float* kept = p.saved + (r * p.f + c);
      x.kept = count >= 4 ? load_kept<true>(kept, plane, 4) : load_kept<false>(kept, plane, count);
#pragma unroll
      for (int k = 0; k < O; ++k)
        x.dy[k] = k < p.o ? to_f32<KIND>(static_cast<const T*>(p.dy)[r * p.ld_y + k]) : 0.0f;
      return x;
    };
    auto use = [&](long r, const Row& x) {
      f4 dh = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int k = 0; k < O; ++k)
          if (O == 1 || k < p.o) dh[e] += x.dy[k] * w[e][k];
      const GateGrad g = gate_grad<false>(p.act, count, dh, x.kept);
      put4<KIND>(static_cast<T*>(p.dg) + r * p.ldh + c, g.dg);
      put4<KIND>(static_cast<T*>(p.du) + r * p.ldh + c, g.du);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int k = 0; k < O; ++k) acc[e][k] += g.h[e] * x.dy[k];
    };
    constexpr int U = O <= 2 ? 4 : 2;  // rows under way
    long r = r0 + slot;
    for (; r + (U - 1) * at_once < r1; r += U * at_once) {
      Row x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = fetch(r + u * at_once);
#pragma unroll
      for (int u = 0; u < U; ++u) use(r + u * at_once, x[u]);
    }
    for (; r < r1; r += at_once) use(r, fetch(r));
  }
  if (!p.partial) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int k = 0; k < O; ++k) part[(threadIdx.x * 4 + e) * O + k] = acc[e][k];
  __syncthreads();
  const int each = p.quads * 4 * O;
  for (int q = threadIdx.x; q < each; q += 256) {
    float v = 0.0f;
    for (int s = 0; s < at_once; ++s) v += part[s * each + q];
    const int col = blockIdx.y * p.quads * 4 + q / O, k = q % O;
    if (col < p.f && k < p.o) p.partial[((long)blockIdx.x * p.f + col) * p.o + k] = v;
  }
}

constexpr int kShares = 32;  // threads that share an entry's slices
template <int KIND>
__global__ __launch_bounds__(256) void k_outs_join(const OutsArgs p) {
  using T = typename ElemOf<KIND>::T;
  constexpr int kEach = 256 / kShares;
  __shared__ float part[kShares][kEach];
  const int share = threadIdx.x / kEach, slot = threadIdx.x % kEach;
  const int entries = p.f * p.o, at = blockIdx.x * kEach + slot;
  float v = 0.0f;
  if (at < entries) {
    const int z1 = p.slices * (share + 1) / kShares;
    int z = p.slices * share / kShares;
    for (; z + 4 <= z1; z += 4) {
      float q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = p.partial[(long)(z + k) * entries + at];
#pragma unroll
      for (int k = 0; k < 4; ++k) v += q[k];
    }
    for (; z < z1; ++z) v += p.partial[(long)z * entries + at];
  }
  part[share][slot] = v;
  __syncthreads();
  if (share || at >= entries) return;
  for (int k = 1; k < kShares; ++k) v += part[k][slot];
  static_cast<T*>(p.dwd)[at / p.o * p.ld_down + at % p.o] = from_f32<KIND>(v);
}

// outputs up to a power of two
int outs_of(int o) { return o <= 1 ? 1 : o <= 2 ? 2 : 4; }

template <class F>
void with_outs(int o, F&& f) {
  switch (outs_of(o)) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 4>{});
  }
}
template <class F>
void with_kind(int elem, F&& f) {
  if (elem == kBf16)
    f(std::integral_constant<int, kBf16>{});
  else if (elem == kF16)
    f(std::integral_constant<int, kF16>{});
  else
    f(std::integral_constant<int, kF32>{});
}

}  // namespace

// (w_down in LDS: up to 32 KB.) A training step, us, these kernels / tiles: 31,920 rows through 70-96-1 in fp32 101 / 116,
// in bf16 70 / 80; 70-96-4 in fp32 105 / 116; in bf16 12,288 rows through 512-240-1 74 / 89, 512-240-4 82 / 89;
// 8,192 through 512-1024-1 136 / 152, 512-1024-4 150 / 152; 131,072 through 2048-240-1 1,086 / 1,170. A
// forward alone in bf16 takes longer, as h is 4 bytes here and 2 as an operand: 26 / 21, 23 / 23, 24 / 23, 35 / 35,
// 37 / 35 and 300 / 288 of these, and has one rounding fewer. Eight outputs were behind in 16 bits
// (w_down's eight reads of LDS an element of h).
bool few_outputs(int d_hidden, int d_out) {
  return d_out <= kFewOutputs && (long)(d_hidden + 7) / 8 * 8 * outs_of(d_out) <= 8192;
}

void run_outs_down(hipStream_t st, int elem, int ncu, const OutsArgs& p) {
  // a row's chunks four a lane where sixteen lanes do for that
  const bool wide = p.ldh * 4 > 16 * 16 * 16;
  const long each = 256 / (wide ? 64 : 16);
  const dim3 grid((unsigned)std::min((p.rows + each - 1) / each, 4l * ncu));
  with_kind(elem, [&](auto kind) {
    with_outs(p.o, [&](auto o) {
      constexpr int K = decltype(kind)::value, O = decltype(o)::value;
      const size_t lds = sizeof(float) * p.ldh * O;
      if (wide)
        hipLaunchKernelGGL((k_outs_down<K, O, 64>), grid, dim3(256), lds, st, p);
      else
        hipLaunchKernelGGL((k_outs_down<K, O, 16>), grid, dim3(256), lds, st, p);
    });
  });
  DPAMD_LAUNCH_CHECK();
}

size_t plan_outs_grad(int ncu, OutsArgs& p) {
  const int all = (int)(p.ldh / 4);
  p.groups = (all + 63) / 64;
  p.quads = (all + p.groups - 1) / p.groups;
  // about four blocks a compute unit, and eight passes over rows a block where there are as many
  const long passes = (p.rows + 256 / p.quads - 1) / (256 / p.quads);
  p.slices = (int)std::max(1l, std::min((passes + 7) / 8, (4l * ncu + p.groups - 1) / p.groups));
  return sizeof(float) * p.slices * (size_t)p.f * p.o;
}

void run_outs_grad(hipStream_t st, int elem, const OutsArgs& p) {
  with_kind(elem, [&](auto kind) {
    constexpr int K = decltype(kind)::value;
    with_outs(p.o, [&](auto o) {
      hipLaunchKernelGGL((k_outs_grad<K, decltype(o)::value>), dim3(p.slices, p.groups), dim3(256), 0, st, p);
    });
    DPAMD_LAUNCH_CHECK();
    if (!p.partial) return;
    const int each = 256 / kShares;
    hipLaunchKernelGGL((k_outs_join<K>), dim3((p.f * p.o + each - 1) / each), dim3(256), 0, st, p);
    DPAMD_LAUNCH_CHECK();
  });
}

}  // namespace dpamd
