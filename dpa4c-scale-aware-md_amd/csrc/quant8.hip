// 8-bit forms of rows: checkpoints of activations (groups of 32 columns, a power of two each), and the
// operands of the 8-bit products (a scale for each token and each output channel).
#include <algorithm>

#include "quant8.h"

namespace dpamd {

namespace {

// (a grid holds fewer than 2^32 threads: the kernels stride over what is beyond)
unsigned grid_of(long blocks) { return (unsigned)std::min(blocks, 1L << 20); }

// ---- checkpoints ------------------------------------------------------------------------
// A group of 32 is held as integers q and the exponent field of its largest magnitude, of which the unit
// is 2^(field - 133): q = x / unit is then below 128, and q * unit is a number of bf16, f16 and fp32 alike (at most
// seven digits), so that what is restored meets the matrix cores of any type without another rounding. A
// scale of max / 127 would halve the error where the maximum is just past a power of two and cost
// that rounding. Field 255 (an infinity or a NaN in the group) restores NaN.
//
// Eight columns a thread, four threads a group: 16-byte loads of 16-bit types, 8-byte stores of q. Bound by
// the bytes: 131,072 x 2048 of bf16 written in 160 us (5.1 TB/s, a copy's rate) and restored in 168.
// Items of a block: ITEMS * 256 consecutive eights of the rows of `per` eights, 256 apart for a thread: four, or
// one where four would leave compute units idle. Row and eight of each by one
// 32-bit division from the block's first.
struct Place {
  long row;
  int c0;
};
__device__ __forceinline__ Place place_of(long base_row, int base_off, int per, int k) {
  const unsigned o = (unsigned)base_off + (unsigned)k, r = o / (unsigned)per;
  return Place{base_row + r, (int)(o - r * (unsigned)per) * 8};
}

template <int KIND, int kItems>
__global__ __launch_bounds__(256) void k_keep8(const KeepArgs p) {
  using T = typename ElemOf<KIND>::T;
  const int wide = p.wide, per = wide / 8;
  const long all = p.rows * per;
  for (long base = (long)blockIdx.x * (kItems * 256); base < all; base += (long)gridDim.x * (kItems * 256)) {
    const long base_row = base / per;
    const int base_off = (int)(base - base_row * per);
    float v[kItems][8];
    Place at[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      at[k] = place_of(base_row, base_off, per, k * 256 + threadIdx.x);
      load8<KIND>(v[k], static_cast<const T*>(p.x) + at[k].row * p.ld + at[k].c0,
                  base + k * 256 + threadIdx.x < all ? p.cols - at[k].c0 : 0);
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(unsigned, v[k][e]) & 0x7fffffffu);
      // (the four threads of a group are four lanes from a multiple of four on: a row is whole groups)
      top = max(top, (unsigned)__shfl_xor((int)top, 1, kWave));
      top = max(top, (unsigned)__shfl_xor((int)top, 2, kWave));
      const int field = (int)(top >> 23);
      unsigned q[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = fminf(fmaxf(ldexpf(v[k][e], 133 - field), -127.0f), 127.0f);
        q[e / 4] |= (field == 255 ? 0u : low_byte(t + kRound)) << (8 * (e % 4));
      }
      if (base + k * 256 + threadIdx.x >= all) continue;
      unsigned long long both = q[0] | (unsigned long long)q[1] << 32;
      *reinterpret_cast<unsigned long long*>(p.kept + at[k].row * wide + at[k].c0) = both;
      if ((at[k].c0 & 31) == 0) p.kept[p.rows * wide + at[k].row * (wide / 32) + at[k].c0 / 32] = (unsigned char)field;
    }
  }
}

// Rows of `cols` columns and zeros up to `cols_out` (a multiple of eight where x is an operand).
template <int KIND, bool ONCE, int kItems>
__global__ __launch_bounds__(256) void k_restore8(const KeepArgs p) {
  using T = typename ElemOf<KIND>::T;
  const int per = (p.cols_out + 7) / 8;
  const long all = p.rows * per;
  T* x = static_cast<T*>(p.out);
  for (long base = (long)blockIdx.x * (kItems * 256); base < all; base += (long)gridDim.x * (kItems * 256)) {
    const long base_row = base / per;
    const int base_off = (int)(base - base_row * per);
    Kept8 v[kItems];
    Place at[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (base + k * 256 + threadIdx.x >= all) continue;
      at[k] = place_of(base_row, base_off, per, k * 256 + threadIdx.x);
      v[k] = load_kept8(p.kept, p.rows, p.wide, at[k].row, at[k].c0);
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (base + k * 256 + threadIdx.x >= all) continue;
      float f[8];
      restore_kept8(v[k], f);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at[k].c0 + e >= p.cols) f[e] = 0.0f;
      store8<KIND, ONCE>(x + at[k].row * p.ld + at[k].c0, f, p.cols_out - at[k].c0);
    }
  }
}

// ---- operands of the 8-bit products -------------------------------------------------------
// A row by T threads of a block (16; 64, a wave; 256), C eights a thread held in registers
// between the maximum and the integers; what is beyond C T eights is read again, from the caches. Zeros up
// to ld_q (a multiple of 16). Bound by the bytes: 16,384 rows of 8192 in bf16 78 us (5.1 TB/s).
template <int KIND, int T, int C>
__global__ __launch_bounds__(256) void k_rows8(const Rows8Args p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int R = 256 / T;
  __shared__ unsigned tops[4];
  const int t = threadIdx.x % T, lane_row = threadIdx.x / T;
  const int eights = (int)(p.ld_q / 8);
  for (long row0 = (long)blockIdx.x * R; row0 < p.rows; row0 += (long)gridDim.x * R) {
    const long row = min(row0 + lane_row, p.rows - 1);  // (the last rows' threads may repeat one)
    const E* x = static_cast<const E*>(p.x) + row * p.ld;
    float v[C][8];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < C; ++k) load8<KIND>(v[k], x + (k * T + t) * 8, p.cols - (k * T + t) * 8);
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(unsigned, v[k][e]) & 0x7fffffffu);
    for (int k = C * T + t; k < eights; k += T) {
      float w[8];
      load8<KIND>(w, x + k * 8, p.cols - k * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(unsigned, w[e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int m = 1; m < (T < 64 ? T : 64); m *= 2) top = max(top, (unsigned)__shfl_xor((int)top, m, kWave));
    if constexpr (T == 256) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
      __syncthreads();
      top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    const RowScale s = row_scale(top);
    if (t == 0) p.scale[row] = s.scale;
    auto put = [&](int k, const float (&w)[8]) {
      if (k >= eights) return;
      *reinterpret_cast<unsigned long long*>(p.q + row * p.ld_q + k * 8) = s.inv == 0.0f ? 0 : quantize8(w, s.inv);
    };
#pragma unroll
    for (int k = 0; k < C; ++k) put(k * T + t, v[k]);
    for (int k = C * T + t; k < eights; k += T) {
      float w[8];
      load8<KIND>(w, x + k * 8, p.cols - k * 8);
      put(k, w);
    }
  }
}

// Weights [d_in][d_out] -> rows of d_in integers, one for each output channel: a block takes 64 channels, finds
// their maxima over all of d_in, and goes over d_in again, 64 at a time through LDS. Done once for a
// served model: nothing here is tuned.
template <int KIND>
__global__ __launch_bounds__(256) void k_weights8(const Weights8Args p) {
  using E = typename ElemOf<KIND>::T;
  __shared__ unsigned tops[4][64];
  __shared__ unsigned char tile[64][68];
  const int c = threadIdx.x & 63, part = threadIdx.x >> 6, col = blockIdx.x * 64 + c;
  const bool in = col < p.d_out;
  const E* w = static_cast<const E*>(p.w) + (in ? col : 0);
  unsigned top = 0;
  for (int k = part; k < p.d_in; k += 4)
    if (in) top = max(top, __builtin_bit_cast(unsigned, to_f32<KIND>(w[k * p.ld_w])) & 0x7fffffffu);
  tops[part][c] = top;
  __syncthreads();
  const RowScale s = row_scale(max(max(tops[0][c], tops[1][c]), max(tops[2][c], tops[3][c])));
  if (in && part == 0) p.scale[col] = s.scale;
  const int whole = (p.d_in + 15) / 16 * 16;  // (what lies between the rows beyond it is the caller's)
  for (int k0 = 0; k0 < whole; k0 += 64) {
    __syncthreads();
    for (int k = part; k < 64; k += 4) {
      const float v = in && k0 + k < p.d_in && s.inv != 0.0f ? to_f32<KIND>(w[(k0 + k) * p.ld_w]) : 0.0f;
      tile[c][k] = (unsigned char)quant8(v, s.inv);
    }
    __syncthreads();
    // 16 threads a channel, four integers each
    for (int r = threadIdx.x / 16; r < 64; r += 16) {
      const int k = (threadIdx.x % 16) * 4;
      if (blockIdx.x * 64 + r < p.d_out && k0 + k < whole)
        *reinterpret_cast<unsigned*>(p.q + (long)(blockIdx.x * 64 + r) * p.ld_q + k0 + k) =
            *reinterpret_cast<const unsigned*>(&tile[r][k]);
    }
  }
}

// four for each thread of a full card (192 x 1600 in fp32: written in 3.8 us with four a thread and 2.9 with one,
// restored in 4.4 and 2.9)
constexpr long kFewEights = 1L << 20;
dim3 blocks_of(long eights, int items) { return dim3(grid_of((eights + items * 256 - 1) / (items * 256))); }

// A row to 16 lanes, to a wave, or to a block: by its length, and few rows to blocks, which are short of loads under way.
// The whole call with 16 output channels, bf16, this form and the other, in us: 100,000 rows of 96 19 and 59 (a wave a
// row), of 384 33 and 62; 500 rows of 2048 11.7 and 12.6 (a wave a row); 60,000 of 1023 52 and 67 (a wave), but
// of 2048 a wave 91 and 16 lanes 115; 40,000 of 4000 125 and 142 (a wave of eight eights a lane) or 148 (a block of
// four a lane); 8,192 of 16,384 112 and 121 (a block of two a lane).
template <int KIND>
void rows_kind(hipStream_t st, const Rows8Args& p) {
  if (p.ld_q <= 16 * 8)
    hipLaunchKernelGGL((k_rows8<KIND, 16, 1>), dim3(grid_of((p.rows + 15) / 16)), dim3(256), 0, st, p);
  else if (p.ld_q <= 16 * 8 * 4 && p.rows > 1024)
    hipLaunchKernelGGL((k_rows8<KIND, 16, 4>), dim3(grid_of((p.rows + 15) / 16)), dim3(256), 0, st, p);
  else if (p.rows <= 1024 && p.ld_q <= 256 * 8)
    hipLaunchKernelGGL((k_rows8<KIND, 256, 1>), dim3(grid_of(p.rows)), dim3(256), 0, st, p);
  else if (p.ld_q <= 16 * 8 * 8 && p.rows > 8192)
    hipLaunchKernelGGL((k_rows8<KIND, 16, 8>), dim3(grid_of((p.rows + 15) / 16)), dim3(256), 0, st, p);
  else if (p.ld_q <= 64 * 8 * 4)
    hipLaunchKernelGGL((k_rows8<KIND, 64, 4>), dim3(grid_of((p.rows + 3) / 4)), dim3(256), 0, st, p);
  else if (p.ld_q <= 256 * 8 * 4)
    hipLaunchKernelGGL((k_rows8<KIND, 256, 2>), dim3(grid_of(p.rows)), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((k_rows8<KIND, 256, 4>), dim3(grid_of(p.rows)), dim3(256), 0, st, p);
}

template <class F>
void by_kind(int elem, F&& f) {
  if (elem == kBf16)
    f(std::integral_constant<int, kBf16>{});
  else if (elem == kF16)
    f(std::integral_constant<int, kF16>{});
  else
    f(std::integral_constant<int, kF32>{});
}

}  // namespace

void keep8(hipStream_t st, int elem, const KeepArgs& p) {
  if (p.rows <= 0) return;
  const long eights = p.rows * (p.wide / 8);
  by_kind(elem, [&](auto k) {
    if (eights < kFewEights)
      hipLaunchKernelGGL((k_keep8<decltype(k)::value, 1>), blocks_of(eights, 1), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((k_keep8<decltype(k)::value, 4>), blocks_of(eights, 4), dim3(256), 0, st, p);
  });
  DPAMD_LAUNCH_CHECK();
}

void restore8(hipStream_t st, int elem, const KeepArgs& p) {
  if (p.rows <= 0) return;
  const long eights = p.rows * ((p.cols_out + 7) / 8);
  const bool once = past_caches(p.rows * p.cols_out * (elem == kF32 ? 4 : 2));
  by_kind(elem, [&](auto k) {
    constexpr int KIND = decltype(k)::value;
    if (once)
      hipLaunchKernelGGL((k_restore8<KIND, true, 4>), blocks_of(eights, 4), dim3(256), 0, st, p);
    else if (eights < kFewEights)
      hipLaunchKernelGGL((k_restore8<KIND, false, 1>), blocks_of(eights, 1), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((k_restore8<KIND, false, 4>), blocks_of(eights, 4), dim3(256), 0, st, p);
  });
  DPAMD_LAUNCH_CHECK();
}

void rows8(hipStream_t st, int elem, const Rows8Args& p) {
  if (p.rows <= 0) return;
  by_kind(elem, [&](auto k) { rows_kind<decltype(k)::value>(st, p); });
  DPAMD_LAUNCH_CHECK();
}

void weights8(hipStream_t st, int elem, const Weights8Args& p) {
  const dim3 grid((p.d_out + 63) / 64);
  by_kind(elem, [&](auto k) { hipLaunchKernelGGL((k_weights8<decltype(k)::value>), grid, dim3(256), 0, st, p); });
  DPAMD_LAUNCH_CHECK();
}

}  // namespace dpamd
