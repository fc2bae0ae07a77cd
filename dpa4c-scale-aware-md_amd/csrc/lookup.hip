// Embedding lookup with scaling and its gradient by sorted ids.
//
// Lookup: out[i] = s E[id_i]. Bytes only: 4 n of ids, the rows that they name, n rows
// written. A row is cut into chunks as wide as its alignment allows (16 bytes at most), lanes side by side on
// a row's chunks, four rows a thread so that their loads are under way together.
//
// Gradient: dE[v] = s sum_{id_i = v} dout_i, without atomics, so that the sums' order is
// fixed by the ids alone. The row indices are sorted by id (stable radix sort, 8 bits a pass;
// ids outside the table sort behind it); then each table row sums its run of the
// sorted rows, and a long run, cut at every kWindow sorted positions, is summed window by
// window first and the windows' sums in order.
#include <algorithm>

#include "kernels.h"
#include "product.h"

namespace dpamd {

namespace {

// ---- elements -------------------------------------------------------------------------
template <int KIND>
struct ElemOf {
  using T = unsigned short;
};
template <>
struct ElemOf<kF32> {
  using T = float;
};

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

// E consecutive elements, loaded and stored as one
template <int KIND, int E>
struct alignas(sizeof(typename ElemOf<KIND>::T) * E) Chunk {
  typename ElemOf<KIND>::T v[E];
};

// ---- lookup ---------------------------------------------------------------------------
constexpr int kLookupRows = 4;  // rows a thread has under way

template <int KIND, int E>
__global__ __launch_bounds__(256) void k_lookup(long n, int vocab, int chunks, int lanes, const int* __restrict__ ids,
                                                const typename ElemOf<KIND>::T* __restrict__ table, long ld_table,
                                                float scale, typename ElemOf<KIND>::T* __restrict__ out, long ld_out) {
  using C = Chunk<KIND, E>;
  const int per = 256 / lanes, sub = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const long step = (long)gridDim.x * per * kLookupRows;
  for (long r0 = ((long)blockIdx.x * per + sub) * kLookupRows; r0 < n; r0 += step) {
    int id[kLookupRows];
#pragma unroll
    for (int k = 0; k < kLookupRows; ++k) {
      id[k] = r0 + k < n ? ids[r0 + k] : -1;
      if (id[k] >= vocab) id[k] = -1;
    }
    for (int c = lane; c < chunks; c += lanes) {
      C v[kLookupRows];
#pragma unroll
      for (int k = 0; k < kLookupRows; ++k) {
        if (id[k] >= 0) {
          v[k] = *reinterpret_cast<const C*>(table + id[k] * ld_table + c * E);
#pragma unroll
          for (int e = 0; e < E; ++e) v[k].v[e] = from_f32<KIND>(to_f32<KIND>(v[k].v[e]) * scale);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) v[k].v[e] = 0;
        }
      }
#pragma unroll
      for (int k = 0; k < kLookupRows; ++k)
        if (r0 + k < n) *reinterpret_cast<C*>(out + (r0 + k) * ld_out + c * E) = v[k];
    }
  }
}

// Elements that a chunk can hold: rows of `width` of both matrices whole chunks, aligned.
template <int KIND>
int chunk_of(int width, const void* a, long lda, const void* b, long ldb) {
  const int size = KIND == kF32 ? 4 : 2;
  for (int e = 16 / size; e > 1; e /= 2)
    if (width % e == 0 && lda % e == 0 && ldb % e == 0 && reinterpret_cast<uintptr_t>(a) % (e * size) == 0 &&
        reinterpret_cast<uintptr_t>(b) % (e * size) == 0)
      return e;
  return 1;
}

template <int KIND, int E>
void launch_lookup(hipStream_t st, long n, int vocab, int width, const int* ids, const void* table, long ld_table,
                   float scale, void* out, long ld_out) {
  using T = typename ElemOf<KIND>::T;
  const int chunks = width / E;
  int lanes = 1;
  while (lanes < chunks && lanes < 256) lanes *= 2;
  const long per = 256 / lanes * kLookupRows;
  const dim3 grid((unsigned)std::min((n + per - 1) / per, 1L << 20));
  hipLaunchKernelGGL((k_lookup<KIND, E>), grid, dim3(256), 0, st, n, vocab, chunks, lanes, ids,
                     static_cast<const T*>(table), ld_table, scale, static_cast<T*>(out), ld_out);
  DPAMD_LAUNCH_CHECK();
}

template <int KIND>
void lookup_kind(hipStream_t st, long n, int vocab, int width, const int* ids, const void* table, long ld_table,
                 float scale, void* out, long ld_out) {
  switch (chunk_of<KIND>(width, table, ld_table, out, ld_out)) {
    case 8:
      if constexpr (KIND != kF32)
        return launch_lookup<KIND, 8>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
    case 4: return launch_lookup<KIND, 4>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
    case 2: return launch_lookup<KIND, 2>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
    default: return launch_lookup<KIND, 1>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
  }
}

// ---- sort -----------------------------------------------------------------------------
constexpr int kSortThreads = 256, kSortWaves = kSortThreads / kWave;
constexpr int kSortItems = 8;                         // a thread
constexpr int kSortTile = kSortThreads * kSortItems;  // a block
constexpr int kBits = 8, kDigits = 1 << kBits;

// The key of row i in the first pass is its id, or vocab where the id is outside the table.
__device__ __forceinline__ unsigned key_of(const int* ids, const unsigned* keys, long i, int vocab) {
  if (keys) return keys[i];
  const int id = ids[i];
  return id >= 0 && id < vocab ? (unsigned)id : (unsigned)vocab;
}

// counts[digit][tile]
__global__ __launch_bounds__(kSortThreads) void k_sort_count(const int* ids, const unsigned* keys, long n, int vocab,
                                                             int shift, int tiles, int* counts) {
  __shared__ int hist[kDigits];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const long base = (long)blockIdx.x * kSortTile;
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const long i = base + k * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(key_of(ids, keys, i, vocab) >> shift) & (kDigits - 1)], 1);
  }
  __syncthreads();
  counts[(long)threadIdx.x * tiles + blockIdx.x] = hist[threadIdx.x];
}

// Places the tile's rows at starts[digit][tile] + rank among the tile's rows of that
// digit, in row order: wave w takes a contiguous run of rows, 64 at a time; the lanes of
// equal digits are found by one ballot a bit.
__global__ __launch_bounds__(kSortThreads) void k_sort_place(const int* ids, const unsigned* keys, const int* rows,
                                                             long n, int vocab, int shift, int tiles,
                                                             const int* starts, unsigned* keys_out, int* rows_out) {
  __shared__ int count[kSortWaves][kDigits];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int w = 0; w < kSortWaves; ++w) count[w][threadIdx.x] = 0;
  __syncthreads();
  const long base = (long)blockIdx.x * kSortTile + wave * (kSortItems * kWave);
  unsigned key[kSortItems];
  int rank[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const long i = base + k * kWave + lane;
    const bool in = i < n;
    key[k] = in ? key_of(ids, keys, i, vocab) : 0u;
    const int digit = (key[k] >> shift) & (kDigits - 1);
    unsigned long long same = __ballot(in);
#pragma unroll
    for (int b = 0; b < kBits; ++b) {
      const bool bit = (digit >> b) & 1;
      const unsigned long long set = __ballot(bit);
      same &= bit ? set : ~set;
    }
    const int below = __popcll(same & ((1ull << lane) - 1));
    if (in) rank[k] = count[wave][digit] + below;
    wave_lds_sync();
    if (in && below == 0) count[wave][digit] += __popcll(same);
    wave_lds_sync();
  }
  __syncthreads();
  {
    int at = starts[(long)threadIdx.x * tiles + blockIdx.x];
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w][threadIdx.x];
      count[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const long i = base + k * kWave + lane;
    if (i < n) {
      const int to = count[wave][(key[k] >> shift) & (kDigits - 1)] + rank[k];
      keys_out[to] = key[k];
      rows_out[to] = rows ? rows[i] : (int)i;
    }
  }
}

// ---- sums of runs ---------------------------------------------------------------------
constexpr int kWindow = 32;   // sorted positions of one window
constexpr int kShort = 64;    // runs up to this length are summed by their table row itself

// first position whose key is >= v
__device__ __forceinline__ int lower_bound(const unsigned* keys, int n, unsigned v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (keys[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// partial[2 w + 0]: the window's part of the run that holds its first position;
// partial[2 w + 1]: of a long run that starts inside it (there is at most one: a run
// longer than a window reaches the window's end). Only for runs longer than kShort. One
// lane sums E columns.
template <int KIND, int E>
__global__ __launch_bounds__(64) void k_grad_windows(int n, int vocab, int chunks, const unsigned* __restrict__ keys,
                                                     const int* __restrict__ rows,
                                                     const typename ElemOf<KIND>::T* __restrict__ dout, long ld,
                                                     float* __restrict__ partial) {
  using C = Chunk<KIND, E>;
  const int w = blockIdx.x, c = blockIdx.y * 64 + threadIdx.x;
  const int b = w * kWindow, e = min(n, b + kWindow);
  const unsigned first = keys[b], last = keys[e - 1];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const unsigned v = part ? last : first;
    if (v >= (unsigned)vocab || (part && last == first)) continue;
    const int lo = lower_bound(keys, n, v), hi = lower_bound(keys, n, v + 1);
    if (hi - lo <= kShort) continue;
    const int from = max(lo, b), to = min(hi, e);
    float acc[E] = {};
    if (c < chunks) {
      for (int i = from; i < to; ++i) {
        const C x = *reinterpret_cast<const C*>(dout + rows[i] * ld + c * E);
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += to_f32<KIND>(x.v[k]);
      }
      float* o = partial + ((long)(2 * w + part) * chunks + c) * E;
#pragma unroll
      for (int k = 0; k < E; ++k) o[k] = acc[k];
    }
  }
}

// One wave a table row and 64 chunks of it.
template <int KIND, int E>
__global__ __launch_bounds__(64) void k_grad_rows(int n, int chunks, const unsigned* __restrict__ keys,
                                                  const int* __restrict__ rows,
                                                  const typename ElemOf<KIND>::T* __restrict__ dout, long ld,
                                                  const float* __restrict__ partial, float scale,
                                                  typename ElemOf<KIND>::T* __restrict__ dtable, long ld_table) {
  using C = Chunk<KIND, E>;
  const int v = blockIdx.x, c = blockIdx.y * 64 + threadIdx.x;
  const int lo = lower_bound(keys, n, v), hi = lower_bound(keys, n, v + 1);
  if (c >= chunks) return;
  float acc[E] = {};
  if (hi - lo <= kShort) {
    for (int i = lo; i < hi; ++i) {
      const C x = *reinterpret_cast<const C*>(dout + rows[i] * ld + c * E);
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] += to_f32<KIND>(x.v[k]);
    }
  } else {
    for (int w = lo / kWindow; w * kWindow < hi; ++w) {
      const int part = lo > w * kWindow;
      const float* p = partial + ((long)(2 * w + part) * chunks + c) * E;
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] += p[k];
    }
  }
  C o;
#pragma unroll
  for (int k = 0; k < E; ++k) o.v[k] = from_f32<KIND>(acc[k] * scale);
  *reinterpret_cast<C*>(dtable + v * ld_table + c * E) = o;
}

struct GradPlan {
  int passes, tiles;
  size_t keys[2], rows[2], counts, starts, scan, partial, bytes;
};

GradPlan grad_plan(long n, int vocab, int width) {
  GradPlan g{};
  int bits = 1;
  while (bits < 31 && (1L << bits) <= vocab) ++bits;  // keys 0 .. vocab
  g.passes = (bits + kBits - 1) / kBits;
  g.tiles = (int)((n + kSortTile - 1) / kSortTile);
  auto take = [&](size_t b) {
    const size_t at = g.bytes;
    g.bytes += (b + 255) & ~size_t(255);
    return at;
  };
  for (int k = 0; k < 2; ++k) {
    g.keys[k] = take(4 * n);
    g.rows[k] = take(4 * n);
  }
  const int m = kDigits * g.tiles;
  g.counts = take(4 * (size_t)m);
  g.starts = take(4 * (size_t)m);
  g.scan = take(scan_temp_bytes(m));
  g.partial = take(8 * ((n + kWindow - 1) / kWindow) * (size_t)width);
  return g;
}

template <int KIND, int E>
void launch_grad(hipStream_t st, long n, int vocab, int width, const void* dout, long ld, float scale, void* dtable,
                 long ld_table, const unsigned* keys, const int* rows, float* partial) {
  using T = typename ElemOf<KIND>::T;
  const int chunks = width / E, cols = (chunks + 63) / 64;
  hipLaunchKernelGGL((k_grad_windows<KIND, E>), dim3((unsigned)((n + kWindow - 1) / kWindow), cols), dim3(64), 0, st,
                     (int)n, vocab, chunks, keys, rows, static_cast<const T*>(dout), ld, partial);
  DPAMD_LAUNCH_CHECK();
  hipLaunchKernelGGL((k_grad_rows<KIND, E>), dim3(vocab, cols), dim3(64), 0, st, (int)n, chunks, keys, rows,
                     static_cast<const T*>(dout), ld, partial, scale, static_cast<T*>(dtable), ld_table);
  DPAMD_LAUNCH_CHECK();
}

template <int KIND>
void grad_kind(hipStream_t st, long n, int vocab, int width, const void* dout, long ld, float scale, void* dtable,
               long ld_table, const unsigned* keys, const int* rows, float* partial) {
  switch (chunk_of<KIND>(width, dout, ld, dtable, ld_table)) {
    case 8:
      if constexpr (KIND != kF32)
        return launch_grad<KIND, 8>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys, rows, partial);
    case 4: return launch_grad<KIND, 4>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys, rows, partial);
    case 2: return launch_grad<KIND, 2>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys, rows, partial);
    default: return launch_grad<KIND, 1>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys, rows, partial);
  }
}

}  // namespace

void lookup_rows(hipStream_t st, int elem, long n, int vocab, int width, const int* ids, const void* table,
                 long ld_table, float scale, void* out, long ld_out) {
  if (elem == kBf16)
    lookup_kind<kBf16>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
  else if (elem == kF16)
    lookup_kind<kF16>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
  else
    lookup_kind<kF32>(st, n, vocab, width, ids, table, ld_table, scale, out, ld_out);
}

size_t lookup_grad_bytes(long n, int vocab, int width) { return grad_plan(n, vocab, width).bytes; }

void lookup_grad(hipStream_t st, int elem, long n, int vocab, int width, const int* ids, const void* dout, long ld,
                 float scale, void* dtable, long ld_table, char* ws) {
  const GradPlan g = grad_plan(n, vocab, width);
  unsigned* keys[2] = {reinterpret_cast<unsigned*>(ws + g.keys[0]), reinterpret_cast<unsigned*>(ws + g.keys[1])};
  int* rows[2] = {reinterpret_cast<int*>(ws + g.rows[0]), reinterpret_cast<int*>(ws + g.rows[1])};
  int* counts = reinterpret_cast<int*>(ws + g.counts);
  int* starts = reinterpret_cast<int*>(ws + g.starts);
  const int m = kDigits * g.tiles;
  for (int p = 0; p < g.passes; ++p) {
    const unsigned* kin = p ? keys[(p + 1) & 1] : nullptr;
    const int* rin = p ? rows[(p + 1) & 1] : nullptr;
    hipLaunchKernelGGL(k_sort_count, dim3(g.tiles), dim3(kSortThreads), 0, st, ids, kin, n, vocab, kBits * p, g.tiles,
                       counts);
    DPAMD_LAUNCH_CHECK();
    exclusive_scan_int(st, counts, starts, m, ws + g.scan, scan_temp_bytes(m));
    hipLaunchKernelGGL(k_sort_place, dim3(g.tiles), dim3(kSortThreads), 0, st, ids, kin, rin, n, vocab, kBits * p,
                       g.tiles, starts, keys[p & 1], rows[p & 1]);
    DPAMD_LAUNCH_CHECK();
  }
  const int last = (g.passes - 1) & 1;
  float* partial = reinterpret_cast<float*>(ws + g.partial);
  if (elem == kBf16)
    grad_kind<kBf16>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys[last], rows[last], partial);
  else if (elem == kF16)
    grad_kind<kF16>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys[last], rows[last], partial);
  else
    grad_kind<kF32>(st, n, vocab, width, dout, ld, scale, dtable, ld_table, keys[last], rows[last], partial);
}

}  // namespace dpamd
