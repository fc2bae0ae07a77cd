// The products of 8-bit integers: tiles of product.h on v_mfma_i32_16x16x64_i8, whose steps hold 128 of k
// and cost what a step of 64 does in 16 bits. 16,384 x 8192 x 2048: 263 us (2,090 TOP/s), matrix cores busy in 0.56 of the
// cycles. Products of few steps are bound by their tiles' ends: a gate of 4,099 x 1023 x 2 x 2737 48 us, 0.24 of the
// cycles.
#include <algorithm>

#include "product.h"

namespace dpamd {

namespace {

using Big = Shape<256, 256, 2, 4>;
using Small = Shape<128, 128, 2, 2>;
using Thin = Shape<64, 128, 1, 4>;
using Tiny = Shape<64, 32, 4, 1>;

// The slices' sums added up as integers, which has no order, and scaled.
template <bool GATE>
__global__ __launch_bounds__(256) void k_join8(const ProductArgs p) {
  constexpr int SUB = GATE ? 2 : 1;
  __shared__ i4 part[SUB][256];
  const int G = p.join, per = 256 / G, quads = p.ldp / 4;
  const int slot = threadIdx.x % per, share = threadIdx.x / per;
  const long at = (long)blockIdx.x * per + slot;
  const bool in = at < (long)p.M * quads;
  const long row = in ? at / quads : 0;
  const int n = in ? (int)(at % quads) * 4 : 0;
  const long plane = (long)p.M * p.ldp, slice = SUB * plane;
  const int* s = reinterpret_cast<const int*>(p.partial) + row * p.ldp + n;
  i4 v[SUB] = {};
  for (int z = p.split * share / G; z < p.split * (share + 1) / G; ++z)
#pragma unroll
    for (int m = 0; m < SUB; ++m) v[m] += *reinterpret_cast<const i4*>(s + z * slice + m * plane);
  if (G > 1) {
#pragma unroll
    for (int m = 0; m < SUB; ++m) part[m][threadIdx.x] = v[m];
    __syncthreads();
    if (share) return;
    for (int k = 1; k < G; ++k)
#pragma unroll
      for (int m = 0; m < SUB; ++m) v[m] += part[m][k * per + slot];
  }
  if (!in) return;
  const int count = p.N - n;
  const f4 col = scales4(p.col_scale[0] + n, count), other = GATE ? scales4(p.col_scale[1] + n, count) : f4{};
  const long to = row * p.ldo[0] + n;
  auto emit = [&](auto kind) {
    constexpr int OUT = decltype(kind)::value;
    const f4 o = scaled4<OUT, GATE>(p.act, __builtin_bit_cast(f4, v[0]), __builtin_bit_cast(f4, v[SUB - 1]),
                                    row_factor(p.row_scale[row]), col, other);
    put_row4<OUT, false>(p.out[0], to, o, count);
  };
  if (p.out_elem == kF32)
    emit(std::integral_constant<int, kF32>{});
  else if (p.out_elem == kF16)
    emit(std::integral_constant<int, kF16>{});
  else
    emit(std::integral_constant<int, kBf16>{});
}

template <bool GATE, class S>
void launch(hipStream_t st, ProductArgs& p) {
  constexpr int SUB = GATE ? 2 : 1;
  p.tiles_m = (p.M + S::BM - 1) / S::BM;
  p.tiles_n = p.tiles_n1 = (p.N + S::BN / SUB - 1) / (S::BN / SUB);
  const long items = (long)p.tiles_m * p.tiles_n * p.split;
  if (items >= 1L << 31) throw HipError{hipErrorInvalidValue, "8-bit product: too many tiles"};
  hipLaunchKernelGGL((k_product<kI8, kRowK, kRowK, GATE ? kEpiScaleGate : kEpiScale, S>),
                     dim3((unsigned)std::min(items, (long)p.blocks)), dim3(S::WM * S::WN * 64), 0, st, p);
  DPAMD_LAUNCH_CHECK();
  if (p.split > 1) {
    const long quads = (long)p.M * (p.ldp / 4);
    p.join = 1;
    while (p.join < 64 && p.split > 8 * p.join && quads * p.join < 1L << 18) p.join *= 2;
    const long per = 256 / p.join;
    hipLaunchKernelGGL((k_join8<GATE>), dim3((unsigned)((quads + per - 1) / per)), dim3(256), 0, st, p);
    DPAMD_LAUNCH_CHECK();
  }
}

template <bool GATE>
void by_shape(hipStream_t st, int shape, ProductArgs& p) {
  if (shape == 0)
    launch<GATE, Big>(st, p);
  else if (shape == 4)
    launch<GATE, Tiny>(st, p);
  else if (shape == 2)
    launch<GATE, Thin>(st, p);
  else
    launch<GATE, Small>(st, p);
}

}  // namespace

void run_product8(hipStream_t st, bool gate, const ProductPlan& plan, ProductArgs& p) {
  p.split = plan.split;
  p.blocks = plan.blocks;
  p.ldp = (p.cols + 3) / 4 * 4;
  p.segs = p.mats = 1;
  if (gate)
    by_shape<true>(st, plan.shape, p);
  else
    by_shape<false>(st, plan.shape, p);
}

}  // namespace dpamd
