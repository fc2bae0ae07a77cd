// Products of 8-bit integers for a few rows (single tokens, a few requests): the weights are read once, from
// memory straight into the operands of v_mfma_i32_16x16x64_i8, 16 output channels by 64 of k in one 16-byte load
// a lane; the rows of x, in fragments of 16, are its other operand. A block takes 16 channels, its waves share
// k and join their integers through LDS, so that no sum leaves the block and all of the weights' loads
// are under way at once. The bytes of the weights bound it: 5.9 us for one row of 2048 -> 8192 (2.8 TB/s, start and end of
// the launch in it; 3.2 at a copy's rate). With more rows each block reads all of them again from L2: 33 rows of
// a gate of 2048 -> 2 x 5000 11.9 us.
#include <algorithm>

#include "quant8.h"

namespace dpamd {

namespace {

constexpr int kStep = 64;   // k of one product
constexpr int kFusedRows = 2;  // (2048 -> 8192: two rows 6.4 us, and four 10.5, where five with a launch of their own take 8.9)
constexpr int kFusedBytes = 48 << 10;

// The 8-bit rows of x in LDS, rows `ld` bytes apart, and their scales: for up to kFusedRows rows each
// block forms them itself (they come from the caches), which saves a launch that the weights would wait for.
// `fetch` issues the weights' loads: after the rows' first ones, as a wait for a load is one for those before it.
template <int KIND, int T, class F>
__device__ __forceinline__ void quantize_rows(const Linear8RowsArgs& p, char* q, int ld, float* scale, unsigned* tops,
                                              F&& fetch) {
  using E = typename ElemOf<KIND>::T;
  const E* x = static_cast<const E*>(p.x);
  const int eights = (p.K + 7) / 8, all = ld / 8;
  // the first kHold eights of a thread stay in registers between the maximum and the integers
  constexpr int kHold = 2;
  float held[kHold][kFusedRows][8];
  unsigned top[kFusedRows] = {};
  auto load = [&](int k, float (&v)[kFusedRows][8]) {
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r)
      if (r < p.rows) load8<KIND>(v[r], x + r * p.ld_x + k * 8, p.K - k * 8);
  };
  auto maximum = [&](const float (&v)[kFusedRows][8]) {
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r)
      if (r < p.rows)
#pragma unroll
        for (int e = 0; e < 8; ++e) top[r] = max(top[r], __builtin_bit_cast(unsigned, v[r][e]) & 0x7fffffffu);
  };
#pragma unroll
  for (int h = 0; h < kHold; ++h) load(h * T + threadIdx.x, held[h]);  // (zeros past the end)
  __builtin_amdgcn_sched_barrier(0);
  fetch();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int h = 0; h < kHold; ++h) maximum(held[h]);
  for (int k = kHold * T + threadIdx.x; k < eights; k += T) {
    float v[kFusedRows][8];
    load(k, v);
    maximum(v);
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2)
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r)
      if (r < p.rows) top[r] = max(top[r], (unsigned)__shfl_xor((int)top[r], m, kWave));
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r) tops[r * (T / 64) + (threadIdx.x >> 6)] = top[r];
  __syncthreads();
  RowScale s[kFusedRows];
#pragma unroll
  for (int r = 0; r < kFusedRows; ++r) {
    unsigned t = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) t = max(t, tops[r * (T / 64) + w]);
    s[r] = row_scale(t);
    if (threadIdx.x == 0) scale[r] = s[r].scale;
  }
  auto put = [&](int k, const float (&v)[kFusedRows][8]) {
    if (k >= all) return;
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r)
      if (r < p.rows)
        *reinterpret_cast<unsigned long long*>(q + r * ld + k * 8) = s[r].inv == 0.0f ? 0 : quantize8(v[r], s[r].inv);
  };
#pragma unroll
  for (int h = 0; h < kHold; ++h) put(h * T + threadIdx.x, held[h]);
  for (int k = kHold * T + threadIdx.x; k < all; k += T) {
    float v[kFusedRows][8];
    load(k, v);
    put(k, v);
  }
  __syncthreads();
}

// F fragments of 16 rows, C of 16 channels (of each matrix); WAVES of a block share k. FUSED: x is quantised
// here (F is 1).
template <int KIND, int F, int C, bool GATE, int WAVES, bool FUSED, int AHEAD>
__global__ __launch_bounds__(64 * WAVES) void k_linear8_rows(const Linear8RowsArgs p) {
  constexpr int MATS = GATE ? 2 : 1, W = MATS * C, T = 64 * WAVES;
  constexpr int kAhead = AHEAD / C;  // steps whose weights are under way
  extern __shared__ __align__(16) char lds[];
  __shared__ float row_scales[kFusedRows];
  __shared__ unsigned tops[kFusedRows * WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.x * (16 * C);
  const int steps = (p.K + kStep - 1) / kStep, s0 = steps * wave / WAVES, s1 = steps * (wave + 1) / WAVES;
  // the lane's rows of weights, and its 16 of the 64 (past the end: the last 16, which meet zeros of x)
  const int last = (p.K + 15) / 16 * 16 - 16;
  const signed char* row_of[W];
#pragma unroll
  for (int m = 0; m < W; ++m) row_of[m] = p.w[m / C] + (long)min(n0 + m % C * 16 + c, p.N - 1) * p.ld_w;
  i4 w[kAhead][W];
  auto weight = [&](int m, int s) {
    return *reinterpret_cast<const i4*>(row_of[m] + min(s * kStep + g * 16, last));
  };
  // (without a test for each step where all of them are there: the tests keep the loads from being issued together)
  auto fetch = [&](int s) {
    if (s + kAhead <= s1) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int m = 0; m < W; ++m) w[u][m] = weight(m, s + u);
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (s + u < s1)
#pragma unroll
          for (int m = 0; m < W; ++m) w[u][m] = weight(m, s + u);
    }
  };
  const int ld = steps * kStep + 16;  // (rows 16 bytes apart in their banks)
  if constexpr (FUSED)
    quantize_rows<KIND, T>(p, lds, ld, row_scales, tops, [&]() { fetch(s0); });
  else
    fetch(s0);

  i4 acc[F][W] = {};
  auto row_part = [&](int f, int s) {  // zeros past k, and for rows past the last
    const int k = s * kStep + g * 16, row = f * 16 + c;
    if (row < p.rows) {
      if constexpr (FUSED) return *reinterpret_cast<const i4*>(lds + row * ld + k);
      if (k <= last) return *reinterpret_cast<const i4*>(p.q + (long)row * p.ld_q + k);
    }
    return i4{0, 0, 0, 0};
  };
  auto multiply = [&](int u, const i4 (&x)[F]) {
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int m = 0; m < W; ++m) acc[f][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][m], x[f], acc[f][m], 0, 0, 0);
  };
  for (int s = s0; s < s1; s += kAhead) {
    if (s + kAhead <= s1) {
      i4 x[kAhead][F];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int f = 0; f < F; ++f) x[u][f] = row_part(f, s + u);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) multiply(u, x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (s + u < s1) {
          i4 x[F];
#pragma unroll
          for (int f = 0; f < F; ++f) x[f] = row_part(f, s + u);
          multiply(u, x);
        }
    }
    fetch(s + kAhead);
  }

  // the waves' sums, joined: a wave finishes the rows of fragment f and channels of fragment h, four channels a lane
  if constexpr (FUSED) __syncthreads();  // (the rows in LDS are read)
  i4* parts = reinterpret_cast<i4*>(lds);
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int m = 0; m < W; ++m) parts[((wave * F + f) * W + m) * 64 + lane] = acc[f][m];
  __syncthreads();
  for (int job = wave; job < F * C; job += WAVES) {
    const int f = job / C, h = job % C;
    const int row = f * 16 + c, n = n0 + h * 16 + 4 * g, count = p.N - n;
    if (row >= p.rows || count <= 0) continue;
    i4 sum[2] = {};
#pragma unroll
    for (int k = 0; k < WAVES; ++k)
#pragma unroll
      for (int m = 0; m < MATS; ++m) sum[m] += parts[((k * F + f) * W + m * C + h) * 64 + lane];
    const f4 col = scales4(p.col_scale[0] + n, count), other = GATE ? scales4(p.col_scale[1] + n, count) : f4{};
    const float scale = FUSED ? row_scales[row % kFusedRows] : p.row_scale[row];
    const f4 v = scaled4<KIND, GATE>(p.act, __builtin_bit_cast(f4, sum[0]), __builtin_bit_cast(f4, sum[1]),
                               row_factor(scale), col, other);
    if (count >= 4)
      put_any4<KIND>(static_cast<typename ElemOf<KIND>::T*>(p.y) + row * p.ld_y + n, v);
    else
      put_row4<KIND, false>(p.y, row * p.ld_y + n, v, count);
  }
}

template <int KIND, int F, int C, bool GATE, int WAVES, bool FUSED>
void launch(hipStream_t st, const Linear8RowsArgs& p) {
  constexpr int kJoin = WAVES * F * C * (GATE ? 2 : 1) * 1024;
  static_assert(kJoin < 64 << 10, "the waves' parts are less than a block's LDS");
  const int steps = (p.K + kStep - 1) / kStep, rows = FUSED ? p.rows * (steps * kStep + 16) : 0;
  const dim3 grid((p.N + 16 * C - 1) / (16 * C)), block(64 * WAVES);
  if (steps >= 8 * WAVES)
    hipLaunchKernelGGL((k_linear8_rows<KIND, F, C, GATE, WAVES, FUSED, 8>), grid, block, std::max(kJoin, rows), st, p);
  else
    hipLaunchKernelGGL((k_linear8_rows<KIND, F, C, GATE, WAVES, FUSED, 4>), grid, block, std::max(kJoin, rows), st, p);
  DPAMD_LAUNCH_CHECK();
}

template <int KIND, bool GATE, int WAVES>
void by_rows(hipStream_t st, const Linear8RowsArgs& p) {
  if (!p.q)
    launch<KIND, 1, 1, GATE, WAVES, true>(st, p);
  else if (p.rows <= 16)
    launch<KIND, 1, 1, GATE, WAVES, false>(st, p);
  else if (!GATE && p.pairs) {
    // two fragments of channels share the rows' loads, as the two matrices of a gate do
    if constexpr (!GATE) {
      if (p.rows <= 32)
        launch<KIND, 2, 2, GATE, 4, false>(st, p);
      else
        launch<KIND, 3, 2, GATE, 4, false>(st, p);
    }
  } else if (p.rows <= 32)
    launch<KIND, 2, 1, GATE, WAVES, false>(st, p);
  else
    launch<KIND, 3, 1, GATE, WAVES, false>(st, p);
}

template <int KIND>
void rows_kind(hipStream_t st, const Linear8RowsArgs& p) {
  if (p.w[1]) {
    if (p.waves == 8)
      by_rows<KIND, true, 8>(st, p);
    else
      by_rows<KIND, true, 4>(st, p);
  } else {
    if (p.waves == 8)
      by_rows<KIND, false, 8>(st, p);
    else
      by_rows<KIND, false, 4>(st, p);
  }
}

}  // namespace

// Whether so many rows are for these kernels, and whether they quantise x themselves. Against tiles, in us: 2048 -> 8192
// 33 rows 12.2 and 15, 48 rows 12.9 and 14.5; but 8192 -> 2048, whose k only waves share here and blocks share there,
// 33 to 48 rows 19 to 21 and 16.3; a gate of 2048 -> 8192 with 64 rows 21.7 and 19.2.
Linear8Form linear8_form(long rows, int K, int N) {
  if (rows > kLinear8Rows || (rows > 32 && K > 2 * N)) return kLinear8Tiles;
  const long ld = (K + kStep - 1) / kStep * kStep + 16;
  return rows <= kFusedRows && rows * ld <= kFusedBytes ? kLinear8Fused : kLinear8FewRows;
}

void run_linear8_rows(hipStream_t st, int elem, int ncu, Linear8RowsArgs& p) {
  const int steps = (p.K + kStep - 1) / kStep, blocks = (p.N + 15) / 16;
  // eight waves where compute units are left over and each wave has eight steps yet: 8192 -> 2048, one row 8.1 us and 10.5
  // with four, 16 rows 13.7 and 14.2; but 4096 -> 4096 16 rows 11.7 and 10.9
  p.waves = blocks < ncu && steps >= 64 ? 8 : 4;
  // 32 channels a block where that leaves a block for each: 2048 -> 8192 33 rows 11.2 us and 11.9, 4096 -> 8192 17.2 and
  // 20.8
  p.pairs = blocks >= 2 * ncu;
  if (elem == kBf16)
    rows_kind<kBf16>(st, p);
  else if (elem == kF16)
    rows_kind<kF16>(st, p);
  else
    rows_kind<kF32>(st, p);
}

}  // namespace dpamd
