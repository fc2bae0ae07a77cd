// The gated block for a few rows (single tokens, single atoms): the weights are read once and
// each element meets up to eight rows, so the bytes bound it; vector units, fp32
// throughout (h is not rounded, as it is from nine rows on; the backward is the same for any number
// of rows, and rounds it), matrices of any alignment.
//
//   k_rows_gate: a block takes 16 bytes by eight lanes of columns (one 128-byte line a
//     row of weights) and a slice of K, 32 rows of weights at a time in 32 lane groups; their sums
//     are joined by shuffles and through LDS, and each slice's go to `partial`.
//   k_rows_down: a block first adds up the slices of g and u that its own slice of
//     d_hidden needs, forms h in LDS, and goes over w_down in the same way.
//   k_rows_join: the slices of y added up.
// Slices are chosen for about four blocks a compute unit, so that enough loads are under
// way; the slices' sums are a few per cent of the weights' bytes.
//
// One row of 2048-8192-2048 in bf16 (101 MB of weights, 22 us at the rate of a copy): 26.7 us, against
// 37 as tile products (13 us of it k_rows_gate, 5.2 TB/s). From nine rows on the tile products
// are ahead: the vector units then take longer than the loads.
#include <algorithm>

#include "product.h"

namespace dpamd {

namespace {

constexpr int kThreads = 256, kColLanes = 8, kRowLanes = kThreads / kColLanes;
constexpr int kMaxSlice = 1024;  // rows of weights a slice: rows * 4 KB of LDS

// elements of 16 bytes
template <int KIND>
constexpr int chunk_of() {
  return KIND == kF32 ? 4 : 8;
}

// N elements at any alignment of the element (the hardware takes unaligned addresses)
template <class T, int N>
struct Some {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ Some<T, N> load_some(const T* p) {
  Some<T, N> s;
  __builtin_memcpy(&s, p, sizeof(s));
  return s;
}

// acc[r][m][e] += sum over the slice's k of x[r][k] w_m[k][c + e]; x in LDS, rows `slice` apart
template <int KIND, int R, int MATS, int E>
__device__ __forceinline__ void sweep(float (&acc)[R][MATS][E], const float* x, int slice, int count,
                                      const typename ElemOf<KIND>::T* const (&w)[MATS], long ld) {
  using T = typename ElemOf<KIND>::T;
  constexpr int U = 4;  // rows of weights under way
  const int first = threadIdx.x / kColLanes;
  int k = first;
  for (; k + (U - 1) * kRowLanes < count; k += U * kRowLanes) {
    Some<T, E> v[U][MATS];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MATS; ++m) v[u][m] = load_some<T, E>(w[m] + (long)(k + u * kRowLanes) * ld);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float a = x[r * slice + k + u * kRowLanes];
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[r][m][e] += a * to_f32<KIND>(v[u][m].v[e]);
      }
  }
  for (; k < count; k += kRowLanes) {
    Some<T, E> v[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) v[m] = load_some<T, E>(w[m] + (long)k * ld);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][m][e] += x[r * slice + k] * to_f32<KIND>(v[m].v[e]);
  }
}

// The 32 lane groups' sums joined (always in the same order) and written: out[r][m][column]
// of this slice; c is the block's first column.
template <int R, int MATS, int E>
__device__ __forceinline__ void join_groups(float (&acc)[R][MATS][E], float* lds, float* out, int rows, int cols,
                                            int c) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cl = threadIdx.x % kColLanes;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float v = acc[r][m][e];
        v += __shfl_xor(v, 8, kWave);
        v = add_xor16(v);
        acc[r][m][e] = add_xor32(v);
      }
  __syncthreads();  // the rows in LDS are read
  if (lane < kColLanes) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int e = 0; e < E; ++e) lds[((wave * R + r) * MATS + m) * kColLanes * E + cl * E + e] = acc[r][m][e];
  }
  __syncthreads();
  constexpr int kEach = R * MATS * kColLanes * E;
  for (int q = threadIdx.x; q < kEach; q += kThreads) {
    const int r = q / (MATS * kColLanes * E), m = q / (kColLanes * E) % MATS, k = q % (kColLanes * E);
    // (the last lanes' columns are moved back to end with the matrix: they repeat sums, equal ones)
    const int at = __builtin_amdgcn_readfirstlane(c) + k / E * E;
    const int col = (at + E <= cols ? at : max(cols - E, 0)) + k % E;
    if (r < rows && col < cols && at < cols)
      out[((long)r * MATS + m) * cols + col] = lds[q] + lds[kEach + q] + lds[2 * kEach + q] + lds[3 * kEach + q];
  }
}

// The lane's first column: whole chunks, the last one moved back to end with the matrix.
__device__ __forceinline__ int column(int block0, int E, int cols) {
  const int c = block0 + (threadIdx.x % kColLanes) * E;
  return c + E <= cols ? c : max(cols - E, 0);
}

template <int KIND, int R, int E>
__global__ __launch_bounds__(kThreads) void k_rows_gate(RowsArgs p) {
  using T = typename ElemOf<KIND>::T;
  extern __shared__ __align__(16) float lds[];
  const int slice = p.slice1, k0 = blockIdx.y * slice, count = min(slice, p.d - k0);
  const T* x = static_cast<const T*>(p.x);
  for (int q = threadIdx.x; q < R * count; q += kThreads) {
    const int r = q / count, k = q % count;
    lds[r * slice + k] = r < p.rows ? to_f32<KIND>(x[r * p.ld_x + k0 + k]) : 0.0f;
  }
  __syncthreads();
  const int block0 = blockIdx.x * kColLanes * E, c = column(block0, E, p.f);
  const T* w[2] = {static_cast<const T*>(p.wg) + k0 * p.ld_hidden + c,
                   static_cast<const T*>(p.wu) + k0 * p.ld_hidden + c};
  float acc[R][2][E] = {};
  sweep<KIND, R, 2, E>(acc, lds, slice, count, w, p.ld_hidden);
  join_groups<R, 2, E>(acc, lds, p.partial1 + (long)blockIdx.y * p.rows * 2 * p.f, p.rows, p.f, block0);
}

template <int KIND, int R, int E>
__global__ __launch_bounds__(kThreads) void k_rows_down(RowsArgs p) {
  using T = typename ElemOf<KIND>::T;
  extern __shared__ __align__(16) float lds[];
  const int slice = p.slice2, k0 = blockIdx.y * slice, count = min(slice, p.f - k0);
  for (int q = threadIdx.x; q < R * count; q += kThreads) {
    const int r = q / count, k = q % count;
    float h = 0.0f;
    if (r < p.rows) {
      const float* s = p.partial1 + (long)r * 2 * p.f + k0 + k;
      const long step = (long)p.rows * 2 * p.f;
      float g = 0.0f, u = 0.0f;
      int z = 0;
      for (; z + 4 <= p.slices1; z += 4) {
        float a[4], b[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) a[y] = s[(z + y) * step], b[y] = s[(z + y) * step + p.f];
#pragma unroll
        for (int y = 0; y < 4; ++y) g += a[y], u += b[y];
      }
      for (; z < p.slices1; ++z) g += s[z * step], u += s[z * step + p.f];
      f4 a, da;
      activate4(p.act, f4{g, g, g, g}, a, da);
      h = a[0] * u;
      if (p.saved && blockIdx.x == 0) {
        p.saved[(long)r * p.f + k0 + k] = g;
        p.saved[(long)(p.rows + r) * p.f + k0 + k] = u;
      }
    }
    lds[r * slice + k] = h;
  }
  __syncthreads();
  const int block0 = blockIdx.x * kColLanes * E, c = column(block0, E, p.o);
  const T* w[1] = {static_cast<const T*>(p.wd) + k0 * p.ld_down + c};
  float acc[R][1][E] = {};
  sweep<KIND, R, 1, E>(acc, lds, slice, count, w, p.ld_down);
  join_groups<R, 1, E>(acc, lds, p.partial2 + (long)blockIdx.y * p.rows * p.o, p.rows, p.o, block0);
}

template <int KIND>
__global__ __launch_bounds__(kThreads) void k_rows_join(RowsArgs p) {
  // eight threads an element, each a contiguous share of the slices, joined in order
  __shared__ float part[kThreads];
  constexpr int G = 8, per = kThreads / G;
  const int slot = threadIdx.x % per, share = threadIdx.x / per;
  const long at = (long)blockIdx.x * per + slot, all = (long)p.rows * p.o;
  const int z0 = p.slices2 * share / G, z1 = p.slices2 * (share + 1) / G;
  float v = 0.0f;
  if (at < all)
    for (int z = z0; z < z1; ++z) v += p.partial2[z * all + at];
  part[threadIdx.x] = v;
  __syncthreads();
  if (share || at >= all) return;
  for (int k = 1; k < G; ++k) v += part[k * per + slot];
  const long to = at / p.o * p.ld_y + at % p.o;
  static_cast<typename ElemOf<KIND>::T*>(p.y)[to] = from_f32<KIND>(v);
}

template <int KIND, int R, int E>
void launch_rows(hipStream_t st, const RowsArgs& p) {
  auto lds = [](int slice, int mats) { return 4 * std::max(R * slice, 4 * R * mats * kColLanes * E); };
  auto blocks = [](int cols) { return (unsigned)((cols + kColLanes * E - 1) / (kColLanes * E)); };
  hipLaunchKernelGGL((k_rows_gate<KIND, R, E>), dim3(blocks(p.f), p.slices1), dim3(kThreads), lds(p.slice1, 2), st, p);
  DPAMD_LAUNCH_CHECK();
  hipLaunchKernelGGL((k_rows_down<KIND, R, E>), dim3(blocks(p.o), p.slices2), dim3(kThreads), lds(p.slice2, 1), st, p);
  DPAMD_LAUNCH_CHECK();
  hipLaunchKernelGGL((k_rows_join<KIND>), dim3((unsigned)(((long)p.rows * p.o + kThreads / 8 - 1) / (kThreads / 8))),
                     dim3(kThreads), 0, st, p);
  DPAMD_LAUNCH_CHECK();
}

template <int KIND, int E>
void rows_by_count(hipStream_t st, const RowsArgs& p) {
  if (p.rows == 1)
    launch_rows<KIND, 1, E>(st, p);
  else if (p.rows == 2)
    launch_rows<KIND, 2, E>(st, p);
  else if (p.rows <= 4)
    launch_rows<KIND, 4, E>(st, p);
  else
    launch_rows<KIND, 8, E>(st, p);
}

template <int KIND>
void rows_kind(hipStream_t st, const RowsArgs& p) {
  constexpr int E = chunk_of<KIND>();
  if (p.f >= E && p.o >= E)
    rows_by_count<KIND, E>(st, p);
  else
    rows_by_count<KIND, 1>(st, p);
}

// slices of K for `cols` columns: about four blocks a compute unit, at least 64 rows of weights each
void slices_of(int K, int cols, int chunk, int ncu, int& slice, int& slices) {
  const int blocks = (cols + kColLanes * chunk - 1) / (kColLanes * chunk);
  int n = std::max(1, std::min(4 * ncu / blocks, K / 64));
  n = std::max(n, (K + kMaxSlice - 1) / kMaxSlice);
  slice = ((K + n - 1) / n + kRowLanes - 1) / kRowLanes * kRowLanes;
  slices = (K + slice - 1) / slice;
}

}  // namespace

size_t plan_rows(int elem, int ncu, RowsArgs& p) {
  const int chunk = elem == kF32 ? 4 : 8, e = p.f >= chunk && p.o >= chunk ? chunk : 1;
  slices_of(p.d, p.f, e, ncu, p.slice1, p.slices1);
  slices_of(p.f, p.o, e, ncu, p.slice2, p.slices2);
  return 4 * ((size_t)p.slices1 * p.rows * 2 * p.f + (size_t)p.slices2 * p.rows * p.o);
}

void run_rows(hipStream_t st, int elem, RowsArgs& p) {
  p.partial2 = p.partial1 + (size_t)p.slices1 * p.rows * 2 * p.f;
  if (elem == kBf16)
    rows_kind<kBf16>(st, p);
  else if (elem == kF16)
    rows_kind<kF16>(st, p);
  else
    rows_kind<kF32>(st, p);
}

}  // namespace dpamd
