// Embedding lookup with scaling and its gradient by sorted ids.
//
// Lookup: out[i] = s E[id_i]. Bytes only: 4 n of ids, the rows that they name, n rows
// written. A row is cut into chunks as wide as its alignment allows (16 bytes at most), lanes side by side on
// a row's chunks, four rows a thread so that their loads are under way together.
//
// Gradient: dE[v] = s sum_{id_i = v} dout_i, without floating-point atomics, so that the sums'
// order does not depend on which block runs first: it is fixed by the ids, the sizes, and the
// alignment of the rows (which sets the chunks, and with them the lanes of a row, the tables of a block and,
// near its limit, the form). It reads n rows, writes vocab rows. Two forms:
//
// Few ids (atom types): a block sums a contiguous share of the rows into tables of its own in
// LDS, one for each row it has under way, so that every entry has one thread; the blocks'
// tables are then added up in order.
//
// Many ids (tokens): the row indices are sorted by id (stable radix sort, 8 bits a pass;
// ids outside the table sort behind it), each table row sums its run of the sorted rows, and
// a long run, cut at every kWindow sorted positions, is summed window by window first and the
// windows' sums in order.
#include <algorithm>

#include "kernels.h"
#include "product.h"

namespace dpamd {

namespace {

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
          v[k] = *reinterpret_cast<const C*>(table + id[k] * ld_table + (long)c * E);
#pragma unroll
          for (int e = 0; e < E; ++e) v[k].v[e] = from_f32<KIND>(to_f32<KIND>(v[k].v[e]) * scale);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) v[k].v[e] = 0;
        }
      }
#pragma unroll
      for (int k = 0; k < kLookupRows; ++k)
        if (r0 + k < n) *reinterpret_cast<C*>(out + (r0 + k) * ld_out + (long)c * E) = v[k];
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

// lanes that read one row
int row_lanes(int chunks) {
  int lanes = 1;
  while (lanes < chunks && lanes < 256) lanes *= 2;
  return lanes;
}

template <int KIND, int E>
void launch_lookup(hipStream_t st, long n, int vocab, int width, const int* ids, const void* table, long ld_table,
                   float scale, void* out, long ld_out) {
  using T = typename ElemOf<KIND>::T;
  const int chunks = width / E, lanes = row_lanes(chunks);
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
constexpr int kSortItems = 4;                         // a thread (8: place 10 to 12 us of 32,768 rows, 4: 7)
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

// Places the tile's rows at starts[digit][tile] (the counts' exclusive sums; null: formed
// here) + rank among the tile's rows of that digit, in row order: wave w takes a contiguous
// run of rows, 64 at a time; the lanes of equal digits are found by one ballot a bit.
__global__ __launch_bounds__(kSortThreads) void k_sort_place(const int* ids, const unsigned* keys, const int* rows,
                                                             long n, int vocab, int shift, int tiles,
                                                             const int* starts, const int* counts,
                                                             unsigned* keys_out, int* rows_out) {
  __shared__ int count[kSortWaves][kDigits];
  __shared__ int totals[kDigits];
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
    int at;
    if (starts) {
      at = starts[(long)threadIdx.x * tiles + blockIdx.x];
    } else {
      // few tiles: this tile's starts from the counts themselves
      int before = 0, total = 0;
#pragma unroll 8
      for (int t = 0; t < tiles; ++t) {
        const int c = counts[(long)threadIdx.x * tiles + t];
        before += t < (int)blockIdx.x ? c : 0;
        total += c;
      }
      int sum = total;  // inclusive over the wave's digits
#pragma unroll
      for (int off = 1; off < kWave; off *= 2) {
        const int v = __shfl_up(sum, off, kWave);
        if (lane >= off) sum += v;
      }
      totals[threadIdx.x] = sum;
      __syncthreads();
      at = before + sum - total;
      for (int w = 0; w < wave; ++w) at += totals[w * kWave + kWave - 1];
    }
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
constexpr int kWindow = 32;     // sorted positions of one window
constexpr int kShort = 64;      // runs up to this length are summed by their table row itself
// Rows up to which one block sorts them all. The whole gradient, tokens among 30,000, 1024 wide in
// bf16, us, one block / tiles: 1,500 43 / 53, 4,000 51 / 58, 8,000 63 / 62.
constexpr int kOneMost = 8192;
constexpr int kScanTiles = 128; // tiles up to which each block of the sort forms its starts itself

// run[2 v], run[2 v + 1]: first position and end of id v's run. Those of ids without rows are
// not written (run_of() tells by the key at the first position).
__device__ __forceinline__ void put_run(const unsigned* keys, int i, int n, int vocab, int* run) {
  const unsigned v = keys[i];
  if (v >= (unsigned)vocab) return;
  if (i == 0 || keys[i - 1] != v) run[2 * (long)v] = i;
  if (i == n - 1 || keys[i + 1] != v) run[2 * (long)v + 1] = i + 1;
}
__device__ __forceinline__ int2 run_of(const unsigned* keys, const int* run, int n, long v) {
  const int lo = run[2 * v];
  if ((unsigned)lo >= (unsigned)n || keys[lo] != (unsigned)v) return int2{0, 0};
  return int2{lo, run[2 * v + 1]};
}
__global__ __launch_bounds__(256) void k_runs(int n, int vocab, const unsigned* __restrict__ keys,
                                              int* __restrict__ run) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) put_run(keys, i, n, vocab, run);
}

// The whole sort and the runs in one block, for up to 1024 ITEMS rows (a launch costs more than
// the work of a pass): as k_sort_place, with the rows in LDS and sixteen waves.
constexpr int kOneWaves = 16, kOneThreads = kOneWaves * kWave;
template <int ITEMS>
__global__ __launch_bounds__(kOneThreads) void k_sort_one(const int* __restrict__ ids, int n, int vocab, int passes,
                                                          unsigned* __restrict__ keys_out, int* __restrict__ rows_out,
                                                          int* __restrict__ run) {
  __shared__ unsigned keys[kOneThreads * ITEMS];
  __shared__ unsigned short rows[kOneThreads * ITEMS];
  __shared__ int count[kOneWaves][kDigits];
  __shared__ int totals[kDigits / kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int i = threadIdx.x; i < n; i += kOneThreads) {
    keys[i] = key_of(ids, nullptr, i, vocab);
    rows[i] = (unsigned short)i;
  }
  for (int p = 0; p < passes; ++p) {
    for (int k = threadIdx.x; k < kOneWaves * kDigits; k += kOneThreads) count[k / kDigits][k % kDigits] = 0;
    __syncthreads();
    unsigned key[ITEMS];
    unsigned short row[ITEMS];
    int rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = (wave * ITEMS + k) * kWave + lane;
      const bool in = i < n;
      key[k] = in ? keys[i] : 0u;
      row[k] = in ? rows[i] : (unsigned short)0;
      rank[k] = 0;
      const int digit = (key[k] >> (kBits * p)) & (kDigits - 1);
      unsigned long long same = __ballot(in);
      if (!same) continue;  // (of the whole wave)
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
    int total = 0, sum = 0;
    if (threadIdx.x < kDigits) {
      for (int w = 0; w < kOneWaves; ++w) total += count[w][threadIdx.x];
      sum = total;
#pragma unroll
      for (int off = 1; off < kWave; off *= 2) {
        const int v = __shfl_up(sum, off, kWave);
        if (lane >= off) sum += v;
      }
      if (lane == kWave - 1) totals[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      int at = sum - total;
      for (int w = 0; w < wave; ++w) at += totals[w];
      for (int w = 0; w < kOneWaves; ++w) {
        const int c = count[w][threadIdx.x];
        count[w][threadIdx.x] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = (wave * ITEMS + k) * kWave + lane;
      if (i < n) {
        const int to = count[wave][(key[k] >> (kBits * p)) & (kDigits - 1)] + rank[k];
        keys[to] = key[k];
        rows[to] = row[k];
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kOneThreads) {
    keys_out[i] = keys[i];
    rows_out[i] = rows[i];
    put_run(keys, i, n, vocab, run);
  }
}

// acc += rows[from .. to) of this lane's chunk, U loads under way
template <int KIND, int E, int U>
__device__ __forceinline__ void add_rows(float (&acc)[E], int from, int to, const int* __restrict__ rows,
                                         const typename ElemOf<KIND>::T* __restrict__ dout, long ld, int c) {
  using C = Chunk<KIND, E>;
  int i = from;
  for (; i + U <= to; i += U) {
    C x[U];
#pragma unroll
    for (int q = 0; q < U; ++q) x[q] = *reinterpret_cast<const C*>(dout + rows[i + q] * ld + (long)c * E);
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] += to_f32<KIND>(x[q].v[k]);
  }
  for (; i < to; ++i) {
    const C x = *reinterpret_cast<const C*>(dout + rows[i] * ld + (long)c * E);
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] += to_f32<KIND>(x.v[k]);
  }
}

// partial[2 w + 0]: the window's part of the run that holds its first position;
// partial[2 w + 1]: of a long run that starts inside it (there is at most one: a run
// longer than a window reaches the window's end). Only for runs longer than kShort.
template <int KIND, int E>
__global__ __launch_bounds__(256) void k_grad_windows(int n, int vocab, int chunks, const unsigned* __restrict__ keys,
                                                      const int* __restrict__ rows, const int* __restrict__ run,
                                                      const typename ElemOf<KIND>::T* __restrict__ dout, long ld,
                                                      float* __restrict__ partial) {
  const int windows = (n + kWindow - 1) / kWindow, lane = threadIdx.x & 63, groups = (chunks + 63) / 64;
  // a wave 64 chunks of a window
  for (long at = (long)blockIdx.x * 4 + threadIdx.x / 64; at < (long)windows * groups; at += (long)gridDim.x * 4) {
    const int w = (int)(at / groups), c = (int)(at % groups) * 64 + lane;
    const int b = w * kWindow, e = min(n, b + kWindow);
    const unsigned first = keys[b], last = keys[e - 1];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const unsigned v = part ? last : first;
      if (v >= (unsigned)vocab || (part && last == first)) continue;
      const int lo = run[2 * (long)v], hi = run[2 * (long)v + 1];  // (v has rows)
      if (hi - lo <= kShort || c >= chunks) continue;
      float acc[E] = {};
      add_rows<KIND, E, 8>(acc, max(lo, b), min(hi, e), rows, dout, ld, c);
      float* o = partial + ((long)(2 * (long)w + part) * chunks + c) * E;
#pragma unroll
      for (int k = 0; k < E; ++k) o[k] = acc[k];
    }
  }
}

// One wave 64 chunks of `each` table rows, whose runs its lanes look up together: several of a large
// table, most of whose rows have none (a wave a row then spends its time on two loads that wait for each
// other: 45 us, with eight 34, of 32,768 tokens among 50,000, 1024 wide in bf16), one of a small table, whose
// rows are long. The runs follow one another in the sorted order; where they hold few rows in all, these are
// loaded before any table row is stored, as a wait for a load is one for the stores before it too: 26 us, for
// 143 MB (with sixteen rows loaded together no faster; a wave for all chunks of its rows instead
// of 64: the gradient of 16,000 tokens among 12,000, 1001 wide, 176 us, so 98).
constexpr int kTogether = 8;
template <int KIND, int E>
__global__ __launch_bounds__(256) void k_grad_rows(int n, int vocab, int chunks, int each,
                                                   const unsigned* __restrict__ keys,
                                                   const int* __restrict__ rows, const int* __restrict__ run,
                                                   const typename ElemOf<KIND>::T* __restrict__ dout, long ld,
                                                   const float* __restrict__ partial, float scale,
                                                   typename ElemOf<KIND>::T* __restrict__ dtable, long ld_table) {
  using C = Chunk<KIND, E>;
  const int lane = threadIdx.x & 63, groups = (chunks + 63) / 64;
  const long parts = (((long)vocab + each - 1) / each) * groups;
  for (long at = (long)blockIdx.x * 4 + threadIdx.x / 64; at < parts; at += (long)gridDim.x * 4) {
    const long v0 = at / groups * each;
    const int c = (int)(at % groups) * 64 + lane, many = (int)min((long)each, vocab - v0);
    const int2 mine = lane < many ? run_of(keys, run, n, v0 + lane) : int2{0, 0};
    auto put = [&](long v, const float (&acc)[E]) {
      C o;
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] = from_f32<KIND>(acc[e] * scale);
      *reinterpret_cast<C*>(dtable + v * ld_table + (long)c * E) = o;
    };
    const unsigned long long with = __ballot(mine.y > mine.x);
    int base = 0, count = 0;
    if (with) {
      base = __builtin_amdgcn_readlane(mine.x, __builtin_ctzll(with));
      count = __builtin_amdgcn_readlane(mine.y, 63 - __builtin_clzll(with)) - base;
    }
    if (count <= kTogether) {
      const int row = lane < count ? rows[base + lane] : 0;
      const int v = lane < count ? (int)keys[base + lane] : -1;
      // (read from the lanes while all of them are under way: those past the chunks hold some of them)
      int from[kTogether], id[kTogether + 1];
#pragma unroll
      for (int q = 0; q < kTogether; ++q) {
        from[q] = __builtin_amdgcn_readlane(row, q);
        id[q] = __builtin_amdgcn_readlane(v, q);
      }
      id[kTogether] = -1;
      if (c < chunks) {
        C x[kTogether];
#pragma unroll
        for (int q = 0; q < kTogether; ++q)
          if (q < count)
            x[q] = *reinterpret_cast<const C*>(dout + from[q] * ld + (long)c * E);
        float acc[E] = {};
        for (int k = 0; k < many; ++k)
          if (!((with >> k) & 1)) put(v0 + k, acc);
#pragma unroll
        for (int q = 0; q < kTogether; ++q)
          if (q < count) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += to_f32<KIND>(x[q].v[e]);
            if (id[q + 1] != id[q]) {
              put(id[q], acc);
#pragma unroll
              for (int e = 0; e < E; ++e) acc[e] = 0.0f;
            }
          }
      }
      continue;
    }
    for (int k = 0; k < many; ++k) {
      const int lo = __builtin_amdgcn_readlane(mine.x, k), hi = __builtin_amdgcn_readlane(mine.y, k);
      if (c >= chunks) continue;
      float acc[E] = {};
      if (hi - lo <= kShort) {
        add_rows<KIND, E, 4>(acc, lo, hi, rows, dout, ld, c);
      } else {
        const int w0 = lo / kWindow, w1 = (hi - 1) / kWindow;
        // the first window's part is the second of that window where the run starts inside it
        const long step = 2 * (long)chunks * E;
        const float* p = partial + ((2 * (long)w0 + (lo > w0 * kWindow)) * chunks + c) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += p[e];
        p = partial + (2 * (long)(w0 + 1) * chunks + c) * E;
        int w = w0 + 1;
        for (; w + 8 <= w1 + 1; w += 8, p += 8 * step) {
          float y[8][E];  // (eight loads under way: a frequent token's run has a hundred windows)
#pragma unroll
          for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) y[q][e] = p[q * step + e];
#pragma unroll
          for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += y[q][e];
        }
        for (; w <= w1; ++w, p += step)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += p[e];
      }
      put(v0 + k, acc);
    }
  }
}

// ---- few ids ----------------------------------------------------------------------------
constexpr int kTableBytes = 64 << 10;  // LDS of a block's tables: two blocks a compute unit
constexpr int kTableRows = 4;          // rows a thread has under way

// The tables of one block: one for each of the 256 / lanes rows that it reads at a time.
// A thread adds its chunks of its rows into its entries, which no other thread touches.
template <int KIND, int E>
__global__ __launch_bounds__(256) void k_grad_tables(long n, int vocab, int chunks, int lanes, long share,
                                                     const int* __restrict__ ids,
                                                     const typename ElemOf<KIND>::T* __restrict__ dout, long ld,
                                                     float* __restrict__ partial) {
  using C = Chunk<KIND, E>;
  extern __shared__ __align__(16) float table[];
  const int per = 256 / lanes, sub = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int entries = vocab * chunks * E;
  for (int k = threadIdx.x; k < per * entries; k += 256) table[k] = 0.0f;
  __syncthreads();
  float* mine = table + sub * entries;
  const long from = blockIdx.x * share, to = min(n, from + share);
  for (long r0 = from + sub; r0 < to; r0 += (long)per * kTableRows) {
    int id[kTableRows];
#pragma unroll
    for (int k = 0; k < kTableRows; ++k) {
      const long r = r0 + (long)k * per;
      id[k] = r < to ? ids[r] : -1;
      if (id[k] >= vocab) id[k] = -1;
    }
    for (int c = lane; c < chunks; c += lanes) {
      C x[kTableRows];
#pragma unroll
      for (int k = 0; k < kTableRows; ++k)
        if (id[k] >= 0) x[k] = *reinterpret_cast<const C*>(dout + (r0 + (long)k * per) * ld + (long)c * E);
#pragma unroll
      for (int k = 0; k < kTableRows; ++k)
        if (id[k] >= 0) {
          float* t = mine + (id[k] * chunks + c) * E;
#pragma unroll
          for (int e = 0; e < E; ++e) t[e] += to_f32<KIND>(x[k].v[e]);
        }
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k < entries; k += 256) {
    float acc = 0.0f;
    for (int q = 0; q < per; ++q) acc += table[q * entries + k];
    partial[(long)blockIdx.x * entries + k] = acc;
  }
}

// The blocks' tables added up: G threads an entry, each a contiguous share of the
// blocks in order, the shares joined in order.
template <int KIND>
__global__ __launch_bounds__(256) void k_grad_join(int blocks, int entries, int width, int G,
                                                   const float* __restrict__ partial, float scale,
                                                   typename ElemOf<KIND>::T* __restrict__ dtable, long ld_table) {
  __shared__ float part[256];
  const int per = 256 / G, slot = threadIdx.x % per, share = threadIdx.x / per;
  const int k = blockIdx.x * per + slot;
  const int b0 = (int)((long)blocks * share / G), b1 = (int)((long)blocks * (share + 1) / G);
  float acc = 0.0f;
  if (k < entries) {
    int b = b0;
    for (; b + 8 <= b1; b += 8) {
      float x[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = partial[(long)(b + q) * entries + k];
#pragma unroll
      for (int q = 0; q < 8; ++q) acc += x[q];
    }
    for (; b < b1; ++b) acc += partial[(long)b * entries + k];
  }
  part[threadIdx.x] = acc;
  __syncthreads();
  if (share || k >= entries) return;
  for (int q = 1; q < G; ++q) acc += part[q * per + slot];
  dtable[k / width * ld_table + k % width] = from_f32<KIND>(acc * scale);
}

// Blocks of the form for few ids, 0 where its tables do not fit. A block has at least
// 16 rows a thread, so that the tables written are few beside the rows read.
int table_blocks(long n, int vocab, int width, int chunks) {
  const long per = 256 / row_lanes(chunks), entries = (long)vocab * width;
  if (per * entries * 4 > kTableBytes) return 0;
  return (int)std::max(1L, std::min(1024L, n / (per * 16)));
}

struct GradPlan {
  int blocks;  // of the form for few ids, or 0
  int passes, tiles;
  size_t keys[2], rows[2], run, counts, starts, scan, partial, bytes;
};

GradPlan grad_plan(long n, int vocab, int width, int chunks) {
  GradPlan g{};
  auto take = [&](size_t b) {
    const size_t at = g.bytes;
    g.bytes += (b + 255) & ~size_t(255);
    return at;
  };
  g.blocks = table_blocks(n, vocab, width, chunks);
  if (g.blocks) {
    g.partial = take(4 * (size_t)g.blocks * vocab * width);
    return g;
  }
  int bits = 1;
  while (bits < 31 && (1L << bits) <= vocab) ++bits;  // keys 0 .. vocab
  g.passes = (bits + kBits - 1) / kBits;
  g.tiles = (int)((n + kSortTile - 1) / kSortTile);
  for (int k = 0; k < 2; ++k) {
    g.keys[k] = take(4 * n);
    g.rows[k] = take(4 * n);
  }
  g.run = take(8 * (size_t)vocab);
  const int m = kDigits * g.tiles;
  g.counts = take(4 * (size_t)m);
  g.starts = take(4 * (size_t)m);
  g.scan = take(scan_temp_bytes(m));
  g.partial = take(8 * ((n + kWindow - 1) / kWindow) * (size_t)width);
  return g;
}

// a grid of `waves` waves in blocks of four, striding where there are more than a launch takes
dim3 wave_blocks(long waves) { return dim3((unsigned)std::min((waves + 3) / 4, 1L << 20)); }

// The rows sorted by id and the ids' runs, in launches over tiles.
void sort_rows(hipStream_t st, const GradPlan& g, long n, int vocab, const int* ids, unsigned* const* keys,
               int* const* rows, int* run, char* ws) {
  int* counts = reinterpret_cast<int*>(ws + g.counts);
  int* starts = g.tiles > kScanTiles ? reinterpret_cast<int*>(ws + g.starts) : nullptr;
  const int m = kDigits * g.tiles;
  for (int p = 0; p < g.passes; ++p) {
    const unsigned* kin = p ? keys[(p + 1) & 1] : nullptr;
    const int* rin = p ? rows[(p + 1) & 1] : nullptr;
    hipLaunchKernelGGL(k_sort_count, dim3(g.tiles), dim3(kSortThreads), 0, st, ids, kin, n, vocab, kBits * p, g.tiles,
                       counts);
    DPAMD_LAUNCH_CHECK();
    if (starts) exclusive_scan_int(st, counts, starts, m, ws + g.scan, scan_temp_bytes(m));
    hipLaunchKernelGGL(k_sort_place, dim3(g.tiles), dim3(kSortThreads), 0, st, ids, kin, rin, n, vocab, kBits * p,
                       g.tiles, starts, counts, keys[p & 1], rows[p & 1]);
    DPAMD_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(k_runs, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (int)n, vocab,
                     keys[(g.passes - 1) & 1], run);
  DPAMD_LAUNCH_CHECK();
}

template <int KIND, int E>
void launch_grad(hipStream_t st, long n, int vocab, int width, const int* ids, const void* dout_, long ld, float scale,
                 void* dtable_, long ld_table, char* ws) {
  using T = typename ElemOf<KIND>::T;
  const T* dout = static_cast<const T*>(dout_);
  T* dtable = static_cast<T*>(dtable_);
  const int chunks = width / E;
  const GradPlan g = grad_plan(n, vocab, width, chunks);
  float* partial = reinterpret_cast<float*>(ws + g.partial);
  if (g.blocks) {
    const int lanes = row_lanes(chunks), entries = vocab * width;
    const long share = (n + g.blocks - 1) / g.blocks;
    hipLaunchKernelGGL((k_grad_tables<KIND, E>), dim3(g.blocks), dim3(256), 256 / lanes * entries * 4, st, n, vocab,
                       chunks, lanes, share, ids, dout, ld, partial);
    DPAMD_LAUNCH_CHECK();
    int G = 1;
    while (G < 256 && g.blocks > 8 * G) G *= 2;
    hipLaunchKernelGGL((k_grad_join<KIND>), dim3((entries + 256 / G - 1) / (256 / G)), dim3(256), 0, st, g.blocks,
                       entries, width, G, partial, scale, dtable, ld_table);
    DPAMD_LAUNCH_CHECK();
    return;
  }
  unsigned* keys[2] = {reinterpret_cast<unsigned*>(ws + g.keys[0]), reinterpret_cast<unsigned*>(ws + g.keys[1])};
  int* rows[2] = {reinterpret_cast<int*>(ws + g.rows[0]), reinterpret_cast<int*>(ws + g.rows[1])};
  int* run = reinterpret_cast<int*>(ws + g.run);
  const unsigned* key = keys[(g.passes - 1) & 1];
  const int* row = rows[(g.passes - 1) & 1];
  if (n <= kOneMost) {
    auto* kernel = n <= kOneThreads ? k_sort_one<1> : n <= 4 * kOneThreads ? k_sort_one<4> : k_sort_one<8>;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(kOneThreads), 0, st, ids, (int)n, vocab, g.passes,
                       keys[(g.passes - 1) & 1], rows[(g.passes - 1) & 1], run);
    DPAMD_LAUNCH_CHECK();
  } else {
    sort_rows(st, g, n, vocab, ids, keys, rows, run, ws);
  }
  if (n > kShort) {  // (else no run is long)
    hipLaunchKernelGGL((k_grad_windows<KIND, E>), wave_blocks((n + kWindow - 1) / kWindow * ((chunks + 63) / 64)), dim3(256), 0, st, (int)n,
                       vocab, chunks, key, row, run, dout, ld, partial);
    DPAMD_LAUNCH_CHECK();
  }
  // Of n tokens among vocab, the gradient in us with 1 / 4 / 8 table rows a wave: 16,000 among 12,000, 1001 wide,
  // 98 / 67 / 64, 1,000 among 12,000, 512 wide, 20 / 18 / 19; 8,000 among 6,000, 1024 wide, 43 / 42 / 42,
  // 20,000 among 2,500, 1024 wide, 50 / 53 / 58; 32,768 among 50,000, 1024 wide, 111 / 85 / 81. (The table's size
  // stands for few rows a table row. Where a large table has many, one is ahead: 500,000 among 20,000, 64
  // wide in fp32, 136 / 142 / 147, 256 wide in bf16, 164 / 171 / 177; 100,000 among them, 60 / 55 / 56.)
  const int each = vocab >= 16384 ? 8 : vocab >= 8192 ? 4 : 1;
  hipLaunchKernelGGL((k_grad_rows<KIND, E>), wave_blocks(((long)vocab + each - 1) / each * ((chunks + 63) / 64)),
                     dim3(256), 0, st, (int)n, vocab, chunks, each, key, row, run, dout, ld, partial, scale, dtable,
                     ld_table);
  DPAMD_LAUNCH_CHECK();
}

template <int KIND>
void grad_kind(hipStream_t st, long n, int vocab, int width, const int* ids, const void* dout, long ld, float scale,
               void* dtable, long ld_table, char* ws) {
  switch (chunk_of<KIND>(width, dout, ld, dtable, ld_table)) {
    case 8:
      if constexpr (KIND != kF32)
        return launch_grad<KIND, 8>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
    case 4: return launch_grad<KIND, 4>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
    case 2: return launch_grad<KIND, 2>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
    default: return launch_grad<KIND, 1>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
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

size_t lookup_grad_bytes(int elem, long n, int vocab, int width, const void* dout, long ld, const void* dtable,
                         long ld_table) {
  const int e = elem == kF32 ? chunk_of<kF32>(width, dout, ld, dtable, ld_table)
                             : chunk_of<kBf16>(width, dout, ld, dtable, ld_table);
  return grad_plan(n, vocab, width, width / e).bytes;
}

void lookup_grad(hipStream_t st, int elem, long n, int vocab, int width, const int* ids, const void* dout, long ld,
                 float scale, void* dtable, long ld_table, char* ws) {
  if (elem == kBf16)
    grad_kind<kBf16>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
  else if (elem == kF16)
    grad_kind<kF16>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
  else
    grad_kind<kF32>(st, n, vocab, width, ids, dout, ld, scale, dtable, ld_table, ws);
}

}  // namespace dpamd
